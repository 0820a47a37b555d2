// The diagonal gated recurrence and its gradient:
//
//   h_t = a_t h_{t-1} + w_t v_t,  a_t = exp(g_t),  o_t = h_t                      per sequence and channel
//   c_t = a_t (do_t + c_{t+1}),  dv_t = w_t (do_t + c_{t+1}),  dw_t = v_t (do_t + c_{t+1}),  dg_t = c_t h_{t-1}
//
// c_t is what flows out of token t into token t - 1; c behind the last token is the final state's gradient, c of the first
// token is the initial state's. A run of tokens acts on the state that enters it as h -> A h + X with A the product of its
// decays, and on the gradient that enters it from behind as c -> A c + Y with the same A; runs compose, so the sequence is
// cut into tiles of 64 tokens whose runs are composed thread by thread, warp by warp and block by block.
//
// What bounds it is HBM: 10 bytes a channel and token forward in 16 bits (v, w, o and the float32 g), 18 backward. So every
// input is read once and every output written once: a block keeps its tile on chip while the runs are composed. At the copy rate an
// SM has 55 instructions to spend on a channel and token, which decides the layout: a warp holds 64 channels, two a lane, and
// eight consecutive tokens, so a lane composes its run alone with packed arithmetic and nothing is shuffled; tiles come by TMA.
// It takes 32 forward and 54 backward (4 x 2048 x 2048, bf16 with a gate). (Eight channels a lane, composed over the warp by shuffles and fed by a thread's own
// asynchronous copies, took 52 forward and was bound by them: 153 us for 4 x 4096 x 2048 channels, bf16, against 59 = 0.86 of the copy
// rate; backward 252 against 100 = 0.92.)
//
// One block walking a sequence would leave most SMs idle (a batch of 2 with 2048 channels is 64 blocks of 64 channels), so a
// cluster of up to 16 blocks takes as many tiles of the same channels at a time: every block sends the run of its tile to the
// others (8 bytes a channel through distributed shared memory, counted by an mbarrier), and each composes what stands before it. The
// order of composition depends on the sizes only: results are the same bits on every run. Blocks' next tiles are on their way
// meanwhile, and several blocks share an SM, because composing is latency: two barriers and the exchange a tile.
//
// The backward pass needs h_{t-1} in float32 (o is rounded, and dg = c h would keep that rounding), so the forward pass of a
// training step leaves the state that enters every 64th token ("marks", 1/16 byte a channel and token) and the backward pass
// composes the 64 tokens of its tile again from there.
#include <algorithm>
#include <cmath>

#include "clusters.cuh"
#include "common.cuh"
#include "tc_utils.cuh"
#include "tensor_map.cuh"

namespace gdn2 {

namespace {

constexpr int kR = 8;               // tokens of a warp
constexpr int kMark = 64;           // tokens between two marks
constexpr int kC = 64;              // channels of a block
constexpr int kMaxCluster = 16;
constexpr int kMaxStages = 4;

struct Tables {                     // packed sequences, the longest first: which each is, its first token, its length, its first mark
  int n;
  int seq[kMaxPacked], tok[kMaxPacked], len[kMaxPacked], mark[kMaxPacked];
};

struct Args {
  const void *v, *w, *dout;
  const float* g;
  void *o, *dv, *dw;
  float *dg, *marks;
  const float* first;               // initial state (forward), gradient of the final state (backward)
  float* last;                      // final state (forward), gradient of the initial state (backward)
  int64_t v_bs, v_ts, w_bs, w_ts, g_bs, g_ts, do_bs, do_ts;    // batch and token strides in elements
  int64_t S;
  int sequences, D, groups;
};
struct __align__(64) Maps {
  CUtensorMap v, w, g, dout;        // [B][S][D] in boxes of a tile
};

// exp(g) for g <= 0. A channel that decays by 1e-3 a token sums thousands of tokens, and there a decay whose error is one-sided by a
// tenth of a 32-bit step shows (expf: 1.2e-5 of the state at a memory of 2000 tokens). So slow decays are a polynomial with one
// rounding at its end (|g| < 1/32: the next term is under 3e-10), the others, whose memory is short, the approximate
// instruction (4 units of 2^-24, and |g| units for its rounded argument). -inf is a decay of 0, NaN stays NaN. Scalar operations
// with immediate constants: packed ones, whose constants take registers or moves, were a third of the kernel's instructions.
__device__ __forceinline__ float decay(float g) {
  float fast;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(fast) : "f"(g * kLog2e));
  const float slow = fmaf(g, fmaf(g, fmaf(g, fmaf(g, 1.f / 24.f, 1.f / 6.f), 0.5f), 1.f), 1.f);
  return fabsf(g) < 0.03125f ? slow : fast;
}
__device__ __forceinline__ float2 decay2(float2 g) { return make_float2(decay(g.x), decay(g.y)); }

// ---------------------------------------------------------------- a lane's two channels

template <typename T> __device__ __forceinline__ float2 lds_pair(uint32_t addr);
template <> __device__ __forceinline__ float2 lds_pair<float>(uint32_t addr) {
  float2 x;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(x.x), "=f"(x.y) : "r"(addr) : "memory");
  return x;
}
template <> __device__ __forceinline__ float2 lds_pair<__nv_bfloat16>(uint32_t addr) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(addr) : "memory");
  return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 lds_pair<__half>(uint32_t addr) {
  uint32_t r;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(addr) : "memory");
  return __half22float2(*reinterpret_cast<const __half2*>(&r));
}
template <typename T> __device__ __forceinline__ void store_pair(T* p, float2 x);
template <> __device__ __forceinline__ void store_pair<float>(float* p, float2 x) { *reinterpret_cast<float2*>(p) = x; }
template <> __device__ __forceinline__ void store_pair<__nv_bfloat16>(__nv_bfloat16* p, float2 x) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x.x, x.y);
}
template <> __device__ __forceinline__ void store_pair<__half>(__half* p, float2 x) {
  *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x.x, x.y);
}

// Where a lane's channels lie. Fed: two neighbours, from a tile in shared memory; not fed (rows that TMA cannot read): 32 apart,
// so that a warp's loads of single elements are whole lines.
// Lanes behind the last channel load the last one over again, so that loads need no branch (with one, a tile's loads went out a few
// at a time: 30 us for 3 x 1001 x 1001 float32 channels), and store nothing.
template <bool Fed> struct Lane {
  int c[2], last;
  bool live[2];
  __device__ __forceinline__ Lane(int group, int lane, int D) {
    c[0] = group * kC + (Fed ? 2 * lane : lane);
    c[1] = c[0] + (Fed ? 1 : 32);
    last = D - 1;
    live[0] = c[0] < D;
    live[1] = c[1] < D;
  }
  template <typename T> __device__ __forceinline__ float2 load(const T* row) const {
    return make_float2(to_f32<T>(row[min(c[0], last)]), to_f32<T>(row[min(c[1], last)]));
  }
  template <typename T> __device__ __forceinline__ void store(T* row, float2 x) const {
    if constexpr (Fed) {
      if (live[0]) store_pair<T>(row + c[0], x);
    } else {
      if (live[0]) row[c[0]] = from_f32<T>(x.x);
      if (live[1]) row[c[1]] = from_f32<T>(x.y);
    }
  }
};

// ---------------------------------------------------------------- runs

struct Run {                       // of a lane's two channels: h -> A h + X
  float2 A, X;
};
__device__ __forceinline__ Run operator*(const Run& later, const Run& first) {
  return Run{fmul2(later.A, first.A), ffma2(later.A, first.X, later.X)};
}
__device__ __forceinline__ Run identity() { return Run{make_float2(1.f, 1.f), make_float2(0.f, 0.f)}; }
__device__ __forceinline__ float4 pack(const Run& r) { return make_float4(r.A.x, r.A.y, r.X.x, r.X.y); }
__device__ __forceinline__ Run unpack(const float4& f) { return Run{make_float2(f.x, f.y), make_float2(f.z, f.w)}; }

// What the blocks of a cluster send one another, double buffered by the parity of the round, and the feed's barriers
template <int W, bool Back> struct Shared {
  float4 runs[W][32], back[Back ? W : 1][32];            // the warps' runs
  float2 entering[32];
  uint64_t bar[2], full[kMaxStages];
  int abort;
};

// By one warp: the run of this block's tile goes to every block of the cluster; returns what enters this tile and moves `carry`
// past the tiles of the whole cluster. Round `it` writes slots that the others read in round it - 2: nobody sends round it before
// its own round it - 1 is complete, which every block entered only after reading round it - 2.
// After a wait that ran out the rounds go on, so that every barrier is met, but what they exchange is arbitrary and their waits end at
// once; it stays in the cluster's shared memory, which no block gives up before it has arrived (after_a_failure).
template <typename Sh>
__device__ __forceinline__ float2 enter_tile(Sh& sh, float4* slots, int64_t it, int rank, int CL, int lane, const Run& run,
                                             float2& carry, uint32_t* status) {
  float2 in = carry;
  if (CL == 1) {
    carry = ffma2(run.A, carry, run.X);
    return in;
  }
  const int p = (int)(it & 1);
  if (lane == 0) tc::mbar_expect_tx(&sh.bar[p], (uint32_t)(CL * 32 * sizeof(float4)));
  __syncwarp();
  float4* mine = slots + (size_t)p * CL * 32 + lane;
  const uint32_t slot = tc::smem_u32(mine + rank * 32), bar = tc::smem_u32(&sh.bar[p]);
  for (int to = 0; to < CL; ++to) {
    uint32_t rslot, rbar;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rslot) : "r"(slot), "r"(to));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rbar) : "r"(bar), "r"(to));
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];"
                 ::"r"(rslot), "f"(run.A.x), "f"(run.A.y), "f"(run.X.x), "f"(run.X.y), "r"(rbar) : "memory");
  }
  if (tc::mbar_wait_warp(&sh.bar[p], (uint32_t)(it >> 1) & 1, &sh.abort, status, 1u << 29)) {
#pragma unroll 4
    for (int r = 0; r < CL; ++r) {
      if (r == rank) in = carry;
      const Run x = unpack(mine[r * 32]);
      carry = ffma2(x.A, carry, x.X);
    }
  }
  return in;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <typename Sh> __device__ __forceinline__ void init_shared(Sh& sh, int CL, int tid) {
  if (tid == 0) {
    sh.abort = 0;
    for (int i = 0; i < 2; ++i) tc::mbar_init(&sh.bar[i], 1);
    for (int i = 0; i < kMaxStages; ++i) tc::mbar_init(&sh.full[i], 1);
    tc::mbar_init_fence();
  }
  if (CL > 1) cluster_sync(); else __syncthreads();
}

struct Place {                     // a block's sequence, channel group and cluster
  int seq, group, rank, CL;
  int64_t batch, start, len, mark;
};
template <bool Packed> __device__ __forceinline__ Place place(const Args& a, const Tables& tb) {
  Place p;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(p.rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(p.CL));
  const int id = blockIdx.x / p.CL;
  p.group = id % a.groups;
  p.seq = id / a.groups;
  if constexpr (Packed) {
    p.batch = 0;
    p.start = tb.tok[p.seq];
    p.len = tb.len[p.seq];
    p.mark = tb.mark[p.seq];
    p.seq = tb.seq[p.seq];
  } else {
    p.batch = p.seq;
    p.start = 0;
    p.len = a.S;
    p.mark = (int64_t)p.seq * ((a.S + kMark - 1) / kMark);
  }
  return p;
}

// ---------------------------------------------------------------- tiles on their way

// A stage holds the rows of g, v, w and dout of a tile, one after the other. What lies behind the sequence's end (another
// sequence's tokens in a packed batch) is never used; what lies outside the tensor comes as zeros.
__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap* map, int c, int t, int b, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
               ::"r"(dst), "l"(map), "r"(c), "r"(t), "r"(b), "r"(bar) : "memory");
}
template <typename T, int W, bool Gate, bool Back> struct Stage {
  static constexpr int kTile = W * kR;
  static constexpr uint32_t kG = kTile * kC * 4, kV = kTile * kC * (uint32_t)sizeof(T);
  static constexpr uint32_t v = kG, w = v + kV, dout = w + (Gate ? kV : 0);
  static constexpr uint32_t bytes = dout + (Back ? kV : 0);
  static __device__ __forceinline__ void fetch(const Maps& m, uint32_t at, uint64_t* full, const Place& p, int64_t t0) {
    const uint32_t bar = tc::smem_u32(full);
    const int c = p.group * kC, t = (int)(p.start + t0), b = (int)p.batch;
    tc::mbar_expect_tx(full, bytes);
    tma_tile(at, &m.g, c, t, b, bar);
    tma_tile(at + v, &m.v, c, t, b, bar);
    if constexpr (Gate) tma_tile(at + w, &m.w, c, t, b, bar);
    if constexpr (Back) tma_tile(at + dout, &m.dout, c, t, b, bar);
  }
};

// ---------------------------------------------------------------- forward

template <typename T, int W, bool Gate, bool Packed, bool Fed>
__global__ void __launch_bounds__(W * 32, W == 8 ? 3 : 1) scan_forward_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args a,
                                                                   const __grid_constant__ Tables tb, int stages, uint32_t* status) {
  using St = Stage<T, W, Gate, false>;
  constexpr int kTile = W * kR;          // tokens of a tile
  extern __shared__ __align__(128) char smem[];
  __shared__ Shared<W, false> sh;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const Place p = place<Packed>(a, tb);
  const Lane<Fed> ch(p.group, lane, a.D);
  float4* slots = reinterpret_cast<float4*>(smem + stages * St::bytes);
  init_shared(sh, p.CL, tid);
  const T* v = static_cast<const T*>(a.v) + p.batch * a.v_bs + p.start * a.v_ts;
  const T* w = Gate ? static_cast<const T*>(a.w) + p.batch * a.w_bs + p.start * a.w_ts : nullptr;
  const float* g = a.g + p.batch * a.g_bs + p.start * a.g_ts;
  T* o = static_cast<T*>(a.o) + (p.batch * a.S + p.start) * a.D;
  float2 carry = make_float2(0.f, 0.f);               // the exchanging warp's: the last, whose run ends the tile
  if (wid == W - 1 && a.first) carry = ch.load(a.first + (int64_t)p.seq * a.D);
  if (wid == W - 1) sh.entering[lane] = carry;        // loaded before the first run is sent: the state may be updated in place by another block

  const int64_t tiles = (p.len + kTile - 1) / kTile, rounds = (tiles + p.CL - 1) / p.CL;
  auto fetch = [&](int64_t it, int s) {               // by one thread
    const int64_t tile = it * p.CL + p.rank;
    if (tile < tiles && !*static_cast<volatile int*>(&sh.abort)) St::fetch(maps, tc::smem_u32(smem) + s * St::bytes, &sh.full[s], p, tile * kTile);
  };
  if constexpr (Fed)
    if (tid == 0)
      for (int s = 0; s < stages; ++s) fetch(s, s);
  int s = 0, phase = 0;
  for (int64_t it = 0; it < rounds; ++it) {
    const int64_t tile = it * p.CL + p.rank, t0 = tile * kTile + wid * kR;
    const int n = p.len - t0 >= kR ? kR : p.len > t0 ? (int)(p.len - t0) : 0;    // this warp's tokens
    float2 dec[kR], x[kR];
    Run run = identity();
    if (n > 0) {
      if constexpr (Fed) {
        // (after a wait that ran out the tile's values are arbitrary, but every barrier is still met)
        if (!tc::mbar_wait_warp(&sh.full[s], phase, &sh.abort, status, 1u << 29)) __syncwarp();
        const uint32_t at = tc::smem_u32(smem) + s * St::bytes;
        const uint32_t row = wid * kR * kC + 2 * lane;
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          dec[r] = lds_pair<float>(at + (row + r * kC) * 4);
          x[r] = lds_pair<T>(at + St::v + (row + r * kC) * (uint32_t)sizeof(T));
          if constexpr (Gate) x[r] = fmul2(x[r], lds_pair<T>(at + St::w + (row + r * kC) * (uint32_t)sizeof(T)));
        }
      } else {
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const int64_t t = t0 + (r < n ? r : 0);
          dec[r] = ch.load(g + t * a.g_ts);
          x[r] = ch.load(v + t * a.v_ts);
          if constexpr (Gate) x[r] = fmul2(x[r], ch.load(w + t * a.w_ts));
        }
      }
#pragma unroll
      for (int r = 0; r < kR; ++r) dec[r] = decay2(dec[r]);
      if (n < kR) {                                   // rows behind the end change nothing
#pragma unroll
        for (int r = 1; r < kR; ++r)
          if (r >= n) { dec[r] = make_float2(1.f, 1.f); x[r] = make_float2(0.f, 0.f); }
      }
      run = Run{dec[0], x[0]};
#pragma unroll
      for (int r = 1; r < kR; ++r) run = Run{dec[r], x[r]} * run;
    }
    sh.runs[wid][lane] = pack(run);
    __syncthreads();
    if constexpr (Fed)
      if (tid == 0) fetch(it + stages, s);            // every warp holds its share of the tile in registers
    Run before = identity();
#pragma unroll
    for (int i = 0; i < W - 1; ++i)
      if (i < wid) before = unpack(sh.runs[i][lane]) * before;
    if (wid == W - 1)
      sh.entering[lane] = enter_tile(sh, slots, it, p.rank, p.CL, lane, run * before, carry, status);
    __syncthreads();
    float2 h = ffma2(before.A, sh.entering[lane], before.X);
    if (a.marks && wid % (kMark / kR) == 0 && n > 0) ch.store(a.marks + (p.mark + t0 / kMark) * a.D, h);
    T* row = o + t0 * a.D;
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      h = ffma2(dec[r], h, x[r]);
      if (r < n) ch.store(row, h);
      row += a.D;
    }
    if (++s >= stages) { s = 0; phase ^= 1; }
  }
  if (a.last && p.rank == 0 && wid == W - 1) ch.store(a.last + (int64_t)p.seq * a.D, carry);
  __syncthreads();
  if (p.CL > 1) cluster_sync();                       // no block leaves while another may still send to it
  tc::after_a_failure(&sh.abort);
}

// ---------------------------------------------------------------- backward

// Tiles the last first: block `rank` of round `it` takes tile tiles - 1 - (it CL + rank).
template <typename T, int W, bool Gate, bool Packed, bool Fed>
__global__ void __launch_bounds__(W * 32, W == 8 ? 2 : 1) scan_backward_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args a,
                                                                    const __grid_constant__ Tables tb, int stages, uint32_t* status) {
  using St = Stage<T, W, Gate, true>;
  constexpr int kTile = W * kR;          // tokens of a tile
  extern __shared__ __align__(128) char smem[];
  __shared__ Shared<W, true> sh;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const Place p = place<Packed>(a, tb);
  const Lane<Fed> ch(p.group, lane, a.D);
  float4* slots = reinterpret_cast<float4*>(smem + stages * St::bytes);
  init_shared(sh, p.CL, tid);
  const T* v = static_cast<const T*>(a.v) + p.batch * a.v_bs + p.start * a.v_ts;
  const T* w = Gate ? static_cast<const T*>(a.w) + p.batch * a.w_bs + p.start * a.w_ts : nullptr;
  const T* dout = static_cast<const T*>(a.dout) + p.batch * a.do_bs + p.start * a.do_ts;
  const float* g = a.g + p.batch * a.g_bs + p.start * a.g_ts;
  const int64_t out0 = (p.batch * a.S + p.start) * a.D;
  float2 carry = make_float2(0.f, 0.f);               // the exchanging warp's: the first, whose run ends the tile from behind
  if (wid == 0 && a.first) carry = ch.load(a.first + (int64_t)p.seq * a.D);
  if (wid == 0) sh.entering[lane] = carry;            // loaded before the first run is sent, as in the forward pass

  const int64_t tiles = (p.len + kTile - 1) / kTile, rounds = (tiles + p.CL - 1) / p.CL;
  auto fetch = [&](int64_t it, int s) {
    const int64_t tile = tiles - 1 - (it * p.CL + p.rank);
    if (tile >= 0 && !*static_cast<volatile int*>(&sh.abort)) St::fetch(maps, tc::smem_u32(smem) + s * St::bytes, &sh.full[s], p, tile * kTile);
  };
  if constexpr (Fed)
    if (tid == 0)
      for (int s = 0; s < stages; ++s) fetch(s, s);
  int s = 0, phase = 0;
  for (int64_t it = 0; it < rounds; ++it) {
    const int64_t tile = tiles - 1 - (it * p.CL + p.rank), t0 = tile * kTile + wid * kR;
    const int n = tile < 0 ? 0 : p.len - t0 >= kR ? kR : p.len > t0 ? (int)(p.len - t0) : 0;
    const uint32_t at = tc::smem_u32(smem) + s * St::bytes, row = wid * kR * kC + 2 * lane;
    auto value = [&](const T* src, int64_t ts, uint32_t part, int r) {
      if constexpr (Fed) return lds_pair<T>(at + part + (row + r * kC) * (uint32_t)sizeof(T));
      else return ch.load(src + (t0 + (r < n ? r : 0)) * ts);
    };
    float2 dec[kR], vv[kR], ww[kR] = {}, dd[kR];
    float2 mark = make_float2(0.f, 0.f);
    if (tile >= 0) mark = ch.load(a.marks + (p.mark + tile * (kTile / kMark)) * a.D);
    Run run = identity(), back = identity();
    if (n > 0) {
      if constexpr (Fed)
        if (!tc::mbar_wait_warp(&sh.full[s], phase, &sh.abort, status, 1u << 29)) __syncwarp();
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        if constexpr (Fed) dec[r] = lds_pair<float>(at + (row + r * kC) * 4);
        else dec[r] = ch.load(g + (t0 + (r < n ? r : 0)) * a.g_ts);
        vv[r] = value(v, a.v_ts, St::v, r);
        if constexpr (Gate) ww[r] = value(w, a.w_ts, St::w, r);
        dd[r] = value(dout, a.do_ts, St::dout, r);
      }
#pragma unroll
      for (int r = 0; r < kR; ++r) dec[r] = decay2(dec[r]);
      if (n < kR) {                                   // rows behind the end change nothing, in either direction
#pragma unroll
        for (int r = 1; r < kR; ++r)
          if (r >= n) {
            dec[r] = make_float2(1.f, 1.f);
            vv[r] = ww[r] = dd[r] = make_float2(0.f, 0.f);
          }
      }
      run = Run{dec[0], Gate ? fmul2(vv[0], ww[0]) : vv[0]};
#pragma unroll
      for (int r = 1; r < kR; ++r) run = Run{dec[r], Gate ? fmul2(vv[r], ww[r]) : vv[r]} * run;
#pragma unroll
      for (int r = kR - 1; r >= 0; --r) {
        const float2 sum = make_float2(back.X.x + dd[r].x, back.X.y + dd[r].y);
        back.X = fmul2(dec[r], sum);
      }
      back.A = run.A;
    }
    sh.runs[wid][lane] = pack(run);
    sh.back[wid][lane] = pack(back);
    __syncthreads();
    if constexpr (Fed)
      if (tid == W * 32 - 1) fetch(it + stages, s); // every warp holds its share of the tile in registers
    Run before = identity(), behind = identity();
#pragma unroll
    for (int i = W - 1; i > 0; --i)
      if (i > wid) behind = unpack(sh.back[i][lane]) * behind;
    if (wid == 0) sh.entering[lane] = enter_tile(sh, slots, it, p.rank, p.CL, lane, back * behind, carry, status);
#pragma unroll
    for (int i = 0; i < W - 1; ++i)
      if (i < wid) before = unpack(sh.runs[i][lane]) * before;
    __syncthreads();
    float2 h = ffma2(before.A, mark, before.X), c = ffma2(behind.A, sh.entering[lane], behind.X);
    if (n > 0) {
      float2 prev[kR];                                // h_{t-1}
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        prev[r] = h;
        h = ffma2(dec[r], h, Gate ? fmul2(vv[r], ww[r]) : vv[r]);
      }
      int64_t e = out0 + (t0 + kR - 1) * a.D;
#pragma unroll
      for (int r = kR - 1; r >= 0; --r) {
        const float2 dh = make_float2(c.x + dd[r].x, c.y + dd[r].y);
        c = fmul2(dec[r], dh);
        if (r < n) {
          ch.store(static_cast<T*>(a.dv) + e, Gate ? fmul2(dh, ww[r]) : dh);
          if constexpr (Gate) ch.store(static_cast<T*>(a.dw) + e, fmul2(dh, vv[r]));
          ch.store(a.dg + e, fmul2(c, prev[r]));
        }
        e -= a.D;
      }
    }
    if (++s >= stages) { s = 0; phase ^= 1; }
  }
  if (a.last && p.rank == 0 && wid == 0) ch.store(a.last + (int64_t)p.seq * a.D, carry);
  __syncthreads();
  if (p.CL > 1) cluster_sync();
  tc::after_a_failure(&sh.abort);
}

// ---------------------------------------------------------------- a thread's VEC neighbouring channels of one token

__device__ __forceinline__ uint4 ld_stream(const void* p) {      // read once
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
  return r;
}
template <typename T, int VEC> struct Piece {                    // 16 bytes of T
  static_assert(VEC * sizeof(T) == 16, "a piece is 16 bytes");
  uint4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = ld_stream(p); }
  __device__ __forceinline__ void get(float (&x)[VEC]) const {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = to_f32<T>(e[i]);
  }
  static __device__ __forceinline__ void store(T* p, const float (&x)[VEC]) {
    uint4 raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = from_f32<T>(x[i]);
    *reinterpret_cast<uint4*>(p) = raw;
  }
};
template <typename T> struct Piece<T, 1> {
  T raw;
  __device__ __forceinline__ void load(const T* p) { raw = *p; }
  __device__ __forceinline__ void get(float (&x)[1]) const { x[0] = to_f32<T>(raw); }
  static __device__ __forceinline__ void store(T* p, const float (&x)[1]) { *p = from_f32<T>(x[0]); }
};
template <int VEC> __device__ __forceinline__ void load_f32(float (&x)[VEC], const float* p) {
  if constexpr (VEC == 1) {
    x[0] = *p;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const uint4 r = ld_stream(p + i);
      x[i] = __uint_as_float(r.x); x[i + 1] = __uint_as_float(r.y);
      x[i + 2] = __uint_as_float(r.z); x[i + 3] = __uint_as_float(r.w);
    }
  }
}
// A state, which the same launch may write: by ordinary loads, not by those for data that nothing writes meanwhile
template <int VEC> __device__ __forceinline__ void load_state(float (&x)[VEC], const float* p) {
  if constexpr (VEC == 1) {
    x[0] = *p;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 r = *reinterpret_cast<const float4*>(p + i);
      x[i] = r.x; x[i + 1] = r.y; x[i + 2] = r.z; x[i + 3] = r.w;
    }
  }
}
template <int VEC> __device__ __forceinline__ void store_f32(float* p, const float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    *p = x[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  }
}
template <int VEC> __device__ __forceinline__ void decays(float (&a)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) a[i] = decay(a[i]);
}

// ---------------------------------------------------------------- few tokens

// Few tokens: a thread takes its channels of a sequence through all of them. The state may be updated in place.
//
// Up to 8 tokens: 0.17 us each beyond the launch, where composing tiles starts at 3.0 us (512 channels of one sequence, bf16: 8 tokens 2.9
// against 3.2, 12 tokens 3.6 against 3.0). Up to 32 where there are many rows, each of which is a block there (256 x 2048 channels: 32
// tokens 23 against 54 us, 64 tokens 54 against 66; 16 x 2048: 16 tokens 4.9 against 5.8, 24 tokens 6.3 against 5.8).
bool few_tokens(int64_t tokens, int64_t rows) { return tokens <= 8 || (tokens <= 32 && tokens <= 8 + rows / 64); }
template <typename T, int VEC, bool Gate>
__global__ void __launch_bounds__(128) scan_steps_kernel(const __grid_constant__ Args a) {
  const int per = (a.D + VEC - 1) / VEC;
  const int64_t id = (int64_t)blockIdx.x * 128 + threadIdx.x, seq = id / per;
  if (seq >= a.sequences) return;
  const int c0 = (int)(id % per) * VEC;
  float h[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) h[i] = 0.f;
  const T* v = static_cast<const T*>(a.v) + seq * a.v_bs + c0;
  const T* w = Gate ? static_cast<const T*>(a.w) + seq * a.w_bs + c0 : nullptr;
  const float* g = a.g + seq * a.g_bs + c0;
  T* o = static_cast<T*>(a.o) + seq * a.S * a.D + c0;
  if (a.first) load_state<VEC>(h, a.first + seq * a.D + c0);
  constexpr int kAhead = 4;                           // tokens in flight
  const int S = (int)a.S;
  for (int t0 = 0; t0 < S; t0 += kAhead) {
    Piece<T, VEC> pv[kAhead], pw[kAhead];
    float dec[kAhead][VEC];
#pragma unroll
    for (int r = 0; r < kAhead; ++r)
      if (t0 + r < S) {
        pv[r].load(v + (t0 + r) * a.v_ts);
        if constexpr (Gate) pw[r].load(w + (t0 + r) * a.w_ts);
        load_f32<VEC>(dec[r], g + (t0 + r) * a.g_ts);
      }
#pragma unroll
    for (int r = 0; r < kAhead; ++r)
      if (t0 + r < S) {
        float x[VEC], wf[VEC];
        decays<VEC>(dec[r]);
        pv[r].get(x);
        if constexpr (Gate) pw[r].get(wf);
#pragma unroll
        for (int i = 0; i < VEC; ++i) h[i] = fmaf(dec[r][i], h[i], Gate ? x[i] * wf[i] : x[i]);
        Piece<T, VEC>::store(o + (int64_t)(t0 + r) * a.D, h);
      }
  }
  if (a.last) store_f32<VEC>(a.last + seq * a.D + c0, h);
}

// ---------------------------------------------------------------- launches

// Clusters of cl blocks that run at one time when per_sm blocks fit on an SM
int places(int per_sm, int cl) {
  static ClusterMemo known[3];
  const void* kernel = reinterpret_cast<const void*>(scan_forward_kernel<__nv_bfloat16, 8, false, false, true>);
  return active_clusters(known[per_sm - 1], kernel, 8 * 32, (size_t)228 * 1024 / per_sm - 1024 - sizeof(Shared<8, false>) - 512, per_sm, cl);
}

// How a scan is laid out: warps of a block, blocks of a cluster, stages of a block's feed: the quickest by this account of it. A
// cluster takes the tiles of its row a round at a time. A round lasts at least as long as the chain of composing and exchanging it,
// and as all that the blocks at work move in it takes at the copy rate (6500 bytes a nanosecond). Rows that find no place wait for
// the next wave; a wave starts and ends in 3 us. Backward, and where sequences are of many lengths, an SM's instructions bound it,
// too, and blocks that share one take their tiles in turn: the busiest SM's where all run at once, the average SM's where they
// follow one another. Measured, bf16 with a gate, in us, forward and backward: chain of one row 0.95 and 1.85 with 8 warps, 1.45 and
// 2.8 with 16 (tiles of twice the tokens); in clusters 0.25 and 0.06 a block more, with 16 warps 0.2 and 0.02; an SM's tile 0.93 and 2.0, with 16
// warps 1.7 and 3.1. Against measurements, backward: 4 x 4096 x 2048 channels, 8 warps in clusters of 2, 16 warps alone: 131, 102 and 129, 100; 16 x 4096 x 1024, 8 warps alone and in
// clusters of 4, 16 warps alone: 259, 224, 203 and 269, 212, 217; forward: 2 x 4096 x 2048, 8 warps, clusters of 1, 2, 4: 64, 44, 33 and
// 65, 44, 32. Packed sequences are of many lengths: the longest alone, all at the copy rate, or all one after another in the
// places there are, whichever is longest (ten of 16037 tokens together, 2048 channels: clusters of 1 88 us, the longest sequence's
// chain; as chosen 61).
struct Layout {
  int warps, cluster, stages;
  size_t smem;
};
Layout layout(int64_t rows, int64_t longest, double average, size_t token_bytes, size_t traffic, bool fed, bool back, int warps_most) {
  Layout best{};
  double least = 0;
  for (int W = 8; W <= warps_most; W *= 2) {
    const int tile = W * kR;
    const size_t stage = fed ? tile * token_bytes : 0;
    const size_t fixed = (size_t)(back ? 2 * W : W + 1) * 512 + 512;          // a block's Shared
    const int64_t tiles = (longest + tile - 1) / tile;
    for (int cl = 1; cl <= kMaxCluster && (cl == 1 || cl <= tiles); cl += cl < kMaxPortableCluster ? 1 : 4) {
      const size_t slots = (size_t)2 * cl * 32 * sizeof(float4);
      for (int per_sm = W > 8 ? 1 : back ? 2 : 3; per_sm >= 1; --per_sm) {     // the kernels' launch bounds, or fewer blocks and more stages
        const size_t room = (size_t)228 * 1024 / per_sm - 1024 - fixed - slots;
        if (room < 2 * stage) continue;
        const int64_t most = places(per_sm, cl);
        const double chain = (back ? (W > 8 ? 2.8 : 1.85) : (W > 8 ? 1.45 : 0.95)) + (cl > 1 ? (W > 8 ? 0.2 + 0.02 * cl : 0.25 + 0.06 * cl) : 0.0) +
                             (fed ? 0.0 : 1.2);
        const int64_t rounds = (tiles + cl - 1) / cl;
        double cost;
        if (average == (double)longest) {
          auto wave = [&](int64_t clusters) {
            const double bytes = (double)clusters * cl * tile * traffic / 6.5e6;
            return clusters == 0 ? 0.0 : rounds * (bytes > chain ? bytes : chain) + 3.0;
          };
          cost = (double)(rows / most) * wave(most) + wave(rows % most);
        } else {                                       // the longest first, and the others after one another in the places that are left
          const double bytes = (double)rows * average * traffic / 6.5e6, mean = average / (tile * cl) + 0.5;
          const double alone = rounds * chain + 3.0, shared = (double)rows / most * (mean * chain + 3.0);
          cost = bytes > alone ? bytes : alone;
          cost = (cost > shared ? cost : shared) + 3.0;
        }
        if (back || average != (double)longest) {
          const double blocks = (double)rows * cl, sms = device_sm_count(), of_tile = back ? (W > 8 ? 3.1 : 2.0) : (W > 8 ? 1.7 : 0.93);
          const double busiest = blocks <= per_sm * sms ? std::ceil(blocks / sms) : blocks / sms;
          const double of_sm = busiest * ((average + tile * cl - 1) / (tile * cl)) * of_tile + 3.0;
          if (of_sm > cost) cost = of_sm;
        }
        if (best.warps == 0 || cost < 0.99 * least) {
          least = cost;
          best.warps = W;
          best.cluster = cl;
          best.stages = fed ? (int)(room / stage) : 0;
          if (best.stages > kMaxStages) best.stages = kMaxStages;
          best.smem = slots + best.stages * stage;
        }
      }
    }
  }
  return best;
}

bool make_map(CUtensorMap* map, const void* p, int size, CUtensorMapDataType type, const Args& a, int tile, int64_t batches, int64_t bs, int64_t ts) {
  const EncodeTiled fn = encode_tiled();
  if (!fn) return false;
  // the stride of a dimension of one entry is never used, but has to be a valid one
  const int64_t row = ((int64_t)a.D * size + 15) / 16 * 16, token = a.S > 1 ? ts * size : row, batch = batches > 1 ? bs * size : token * a.S;
  const cuuint64_t dims[3] = {(cuuint64_t)a.D, (cuuint64_t)a.S, (cuuint64_t)batches}, strides[2] = {(cuuint64_t)token, (cuuint64_t)batch};
  const cuuint32_t box[3] = {kC, (cuuint32_t)tile, 1}, unit[3] = {1, 1, 1};
  return fn(map, type, 3, const_cast<void*>(p), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
template <typename T> constexpr CUtensorMapDataType map_type() {
  return sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;   // copied as they are
}

template <typename T, bool Gate, bool Packed, bool Fed>
int launch_scan(const Args& a0, const Tables& tb, int64_t longest, double average, bool backward, cudaStream_t st) {
  Args a = a0;
  a.groups = (a.D + kC - 1) / kC;
  const int64_t rows = (int64_t)a.sequences * a.groups, batches = Packed ? 1 : a.sequences;
  const size_t token = kC * (4 + sizeof(T) * (1 + Gate + backward));                                   // read
  const size_t written = kC * (backward ? 4 + sizeof(T) * (1 + Gate) : sizeof(T));
  const Layout l = layout(rows, longest, average, token, token + written, Fed, backward, Fed ? 16 : 8);
  if (rows * l.cluster > 2147483647LL) return GDN2_ERR_BAD_SHAPE;
  Maps maps{};
  const int tile = l.warps * kR;
  if (Fed && (!make_map(&maps.v, a.v, sizeof(T), map_type<T>(), a, tile, batches, a.v_bs, a.v_ts) ||
              !make_map(&maps.g, a.g, 4, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, a, tile, batches, a.g_bs, a.g_ts) ||
              (Gate && !make_map(&maps.w, a.w, sizeof(T), map_type<T>(), a, tile, batches, a.w_bs, a.w_ts)) ||
              (backward && !make_map(&maps.dout, a.dout, sizeof(T), map_type<T>(), a, tile, batches, a.do_bs, a.do_ts))))
    return GDN2_ERR_UNSUPPORTED;
  uint32_t* status = device_status_word();
  if (!status) return record_cuda_error(cudaGetLastError());
  auto kernel = backward ? scan_backward_kernel<T, 8, Gate, Packed, Fed> : scan_forward_kernel<T, 8, Gate, Packed, Fed>;
  if constexpr (Fed)
    if (l.warps > 8) kernel = backward ? scan_backward_kernel<T, 16, Gate, Packed, true> : scan_forward_kernel<T, 16, Gate, Packed, true>;
  GDN2_CUDA_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), l.smem));
  if (l.cluster > kMaxPortableCluster) GDN2_CUDA_TRY(allow_large_clusters(reinterpret_cast<const void*>(kernel)));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = l.cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * l.cluster));
  cfg.blockDim = dim3(l.warps * 32);
  cfg.dynamicSmemBytes = l.smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  GDN2_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, maps, a, tb, l.stages, status));
  return GDN2_OK;
}

// Rows that no tensor map can describe are loaded by the threads
template <typename T, bool Gate, bool Packed, bool Fed>
int launch_any(const Args& a, const Tables& tb, int64_t longest, double average, bool backward, cudaStream_t st) {
  const int rc = launch_scan<T, Gate, Packed, Fed>(a, tb, longest, average, backward, st);
  if constexpr (Fed)
    if (rc == GDN2_ERR_UNSUPPORTED) return launch_scan<T, Gate, Packed, false>(a, tb, longest, average, backward, st);
  return rc;
}

template <typename T, int VEC, bool Gate>
int launch_all(const Args& a, const int64_t* cu, bool backward, cudaStream_t st) {
  if (!cu) {
    Tables none;
    none.n = 0;
    if (!backward && few_tokens(a.S, (int64_t)a.sequences * ((a.D + kC - 1) / kC)) && !a.marks) {
      const int64_t threads = (int64_t)a.sequences * ((a.D + VEC - 1) / VEC), blocks = (threads + 127) / 128;
      if (blocks > 2147483647LL) return GDN2_ERR_BAD_SHAPE;
      scan_steps_kernel<T, VEC, Gate><<<(unsigned)blocks, 128, 0, st>>>(a);
      GDN2_CUDA_TRY(cudaGetLastError());
      return GDN2_OK;
    }
    return launch_any<T, Gate, false, (VEC > 1)>(a, none, a.S, (double)a.S, backward, st);
  }
  int64_t mark = 0;
  for (int i0 = 0; i0 < a.sequences; i0 += kMaxPacked) {
    Tables tb;
    tb.n = a.sequences - i0 < kMaxPacked ? a.sequences - i0 : kMaxPacked;
    int order[kMaxPacked], marks[kMaxPacked];
    for (int i = 0; i < tb.n; ++i) {
      order[i] = i;
      marks[i] = (int)mark;
      mark += (cu[i0 + i + 1] - cu[i0 + i] + kMark - 1) / kMark;
    }
    auto len = [&](int i) { return cu[i0 + i + 1] - cu[i0 + i]; };
    std::sort(order, order + tb.n, [&](int x, int y) { return len(x) != len(y) ? len(x) > len(y) : x < y; });
    for (int k = 0; k < tb.n; ++k) {
      const int i = order[k];
      tb.seq[k] = i;
      tb.tok[k] = (int)cu[i0 + i];
      tb.len[k] = (int)len(i);
      tb.mark[k] = marks[i];
    }
    const int64_t longest = len(order[0]);
    const double average = (double)(cu[i0 + tb.n] - cu[i0]) / tb.n;
    Args part = a;
    part.sequences = tb.n;
    if (a.first) part.first = a.first + (int64_t)i0 * a.D;
    if (a.last) part.last = a.last + (int64_t)i0 * a.D;
    const int rc = launch_any<T, Gate, true, (VEC > 1)>(part, tb, longest, average, backward, st);
    if (rc != GDN2_OK) return rc;
  }
  return GDN2_OK;
}

template <typename T>
int dispatch(const Args& a, const int64_t* cu, bool wide, bool backward, cudaStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  if (wide) return a.w ? launch_all<T, V, true>(a, cu, backward, st) : launch_all<T, V, false>(a, cu, backward, st);
  return a.w ? launch_all<T, 1, true>(a, cu, backward, st) : launch_all<T, 1, false>(a, cu, backward, st);
}

int check(const gdn2_recurrence_args& r, int dtype, bool backward) {
  if (dtype != GDN2_F32 && dtype != GDN2_BF16 && dtype != GDN2_F16) return GDN2_ERR_BAD_DTYPE;
  if (r.B <= 0 || r.S <= 0 || r.D <= 0 || r.B > (1 << 30) || r.S > (1LL << 30) || r.D > (1 << 24)) return GDN2_ERR_BAD_SHAPE;
  if (!r.v || !r.g || (backward ? !r.dout || !r.dv || !r.dg || !r.marks || (r.w && !r.dw) : !r.o)) return GDN2_ERR_NULL_POINTER;
  if (r.v_token_stride < 0 || r.g_token_stride < 0 || r.v_batch_stride < 0 || r.g_batch_stride < 0 || r.w_token_stride < 0 ||
      r.w_batch_stride < 0 || r.do_token_stride < 0 || r.do_batch_stride < 0)
    return GDN2_ERR_BAD_SHAPE;
  if (r.cu_seqlens) {
    if (r.B != 1 || r.sequences <= 0 || r.sequences > (1 << 30) || r.cu_seqlens[0] != 0 || r.cu_seqlens[r.sequences] != r.S)
      return GDN2_ERR_BAD_SHAPE;
    for (int64_t i = 0; i < r.sequences; ++i)
      if (r.cu_seqlens[i + 1] < r.cu_seqlens[i]) return GDN2_ERR_BAD_SHAPE;
  }
  return GDN2_OK;
}

// TMA and 16-byte pieces need rows that start on 16 bytes, pieces a number of channels that they divide; a dimension that is not
// materialised (stride 0) is not one TMA can walk
bool all_wide(const gdn2_recurrence_args& r, int dtype, bool backward) {
  const int64_t esz = dtype == GDN2_F32 ? 4 : 2, V = 16 / esz;
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  auto rows = [&](const void* p, int64_t bs, int64_t ts, int64_t size) {
    return !p || (aligned(p) && bs * size % 16 == 0 && ts * size % 16 == 0 && (r.B == 1 || bs > 0) && (r.S == 1 || ts > 0) &&
                  bs * size < (1LL << 40) && ts * size < (1LL << 40));
  };
  if (r.D % V) return false;
  if (!rows(r.v, r.v_batch_stride, r.v_token_stride, esz) || !rows(r.g, r.g_batch_stride, r.g_token_stride, 4) ||
      !rows(r.w, r.w_batch_stride, r.w_token_stride, esz) || !aligned(r.state) || !aligned(r.final_state) || !aligned(r.marks))
    return false;
  if (!backward) return aligned(r.o);
  return rows(r.dout, r.do_batch_stride, r.do_token_stride, esz) && aligned(r.dv) && aligned(r.dw) && aligned(r.dg) && aligned(r.dstate);
}

int run(const gdn2_recurrence_args& r, int dtype, bool backward, cudaStream_t st) {
  int rc = check(r, dtype, backward);
  if (rc == GDN2_OK) rc = own_context();
  if (rc != GDN2_OK) return rc;
  Args a{};
  a.v = r.v; a.w = r.w; a.g = r.g; a.o = r.o; a.marks = r.marks;
  a.first = r.state; a.last = r.final_state;
  a.v_bs = r.v_batch_stride; a.v_ts = r.v_token_stride;
  a.w_bs = r.w_batch_stride; a.w_ts = r.w_token_stride;
  a.g_bs = r.g_batch_stride; a.g_ts = r.g_token_stride;
  a.S = r.S;
  a.D = (int)r.D;
  a.sequences = (int)(r.cu_seqlens ? r.sequences : r.B);
  if (backward) {
    a.dout = r.dout; a.dv = r.dv; a.dw = r.dw; a.dg = r.dg;
    a.do_bs = r.do_batch_stride; a.do_ts = r.do_token_stride;
    a.first = r.dfinal_state; a.last = r.dstate;
  }
  const bool wide = all_wide(r, dtype, backward);
  if (dtype == GDN2_BF16) return dispatch<__nv_bfloat16>(a, r.cu_seqlens, wide, backward, st);
  if (dtype == GDN2_F16) return dispatch<__half>(a, r.cu_seqlens, wide, backward, st);
  return dispatch<float>(a, r.cu_seqlens, wide, backward, st);
}

}  // namespace
}  // namespace gdn2

extern "C" {

size_t gdn2_recurrence_marks(int64_t B, int64_t S, const int64_t* cu_seqlens, int64_t sequences) {
  const int64_t m = gdn2::kMark;
  if (!cu_seqlens) return (size_t)(B * ((S + m - 1) / m));
  int64_t n = 0;
  for (int64_t i = 0; i < sequences; ++i) n += (cu_seqlens[i + 1] - cu_seqlens[i] + m - 1) / m;
  return (size_t)n;
}

int gdn2_recurrence_forward(const gdn2_recurrence_args* args, int dtype, void* stream) {
  if (!args) return GDN2_ERR_NULL_POINTER;
  return gdn2::run(*args, dtype, false, static_cast<cudaStream_t>(stream));
}

int gdn2_recurrence_backward(const gdn2_recurrence_args* args, int dtype, void* stream) {
  if (!args) return GDN2_ERR_NULL_POINTER;
  return gdn2::run(*args, dtype, true, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
