// The diagonal gated recurrence and its gradient:
//
//   h_t = a_t h_{t-1} + w_t v_t,  a_t = exp(g_t),  o_t = h_t                      per sequence and channel
//   c_t = a_t (do_t + c_{t+1}),  dv_t = w_t (do_t + c_{t+1}),  dw_t = v_t (do_t + c_{t+1}),  dg_t = c_t h_{t-1}
//
// c_t is what flows out of token t into token t - 1; c behind the last token is the final state's gradient, c of the first
// token is the initial state's. A run of tokens acts on the state that enters it as h -> A h + X with A the product of its
// decays, and on the gradient that enters it from behind as c -> A c + Y with the same A; runs compose, so the sequence is
// cut into tiles whose runs are composed thread by thread, warp by warp and block by block.
//
// What bounds it is HBM: 10 bytes a channel and token forward in 16 bits (v, w, o and the float32 g), 18 backward, against
// some 30 instructions. So every input is read once and every output written once: a block keeps its tile in registers while
// the tiles' runs are composed. One block walking a sequence would leave most SMs idle (a batch of 2 with 2048 channels is 64
// blocks of 64 channels), so a cluster of up to 8 blocks takes 8 tiles of the same channels at a time: every block sends the
// run of its tile to the others (8 bytes a channel through distributed shared memory, counted by an mbarrier), and each composes
// what stands before it. The order of composition depends on the sizes only: results are the same bits on every run.
//
// The backward pass needs h_{t-1} in float32 (o is rounded, and dg = c h would keep that rounding), so the forward pass of a
// training step leaves the state that enters every 64th token ("marks", 1/16 byte a channel and token) and the backward pass
// composes the 64 tokens of its tile again from there.
#include <cooperative_groups.h>

#include "common.cuh"
#include "tc_utils.cuh"

namespace gdn2 {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMarkTokens = 64;     // tokens between two marks, and of a backward tile
constexpr int kMaxCluster = 8;
constexpr int kStepTokens = 8;      // calls of at most so many tokens go token by token

struct Tables {                     // packed sequences: first token and first mark of each
  int n;
  int tok[kMaxPacked + 1];
  int mark[kMaxPacked + 1];
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

// exp(g) for g <= 0 with one rounding behind a polynomial: 2^n (1 + p), p the Taylor polynomial of exp(r) - 1 up to r^7 on
// |r| <= log(2) / 2 (remainder 5e-9). Channels that decay by 1e-3 a token sum thousands of tokens, and there a decay whose
// error is one-sided by a tenth of a 32-bit step shows (expf: 1.2e-5 of the state at a memory of 2000 tokens).
// g under -100 is a decay of 0, -inf among them; NaN stays NaN.
__device__ __forceinline__ float2 decay2(float2 g) {
  g.x = g.x < -100.f ? -100.f : g.x;
  g.y = g.y < -100.f ? -100.f : g.y;
  const float magic = 12582912.f;   // 1.5 * 2^23: adding it rounds to an integer
  const float2 one = make_float2(1.f, 1.f);
  const float2 t = ffma2(g, make_float2(kLog2e, kLog2e), make_float2(magic, magic));
  const float2 n = ffma2(t, one, make_float2(-magic, -magic));
  float2 r = ffma2(n, make_float2(-0.693359375f, -0.693359375f), g);             // log(2) in two parts: the first has 10 bits,
  r = ffma2(n, make_float2(2.12194440e-4f, 2.12194440e-4f), r);                   // so its product with n is exact
  auto c = [](float x) { return make_float2(x, x); };
  float2 q = ffma2(r, c(1.f / 5040.f), c(1.f / 720.f));
  q = ffma2(r, q, c(1.f / 120.f));
  q = ffma2(r, q, c(1.f / 24.f));
  q = ffma2(r, q, c(1.f / 6.f));
  q = ffma2(r, q, c(0.5f));
  const float2 p = ffma2(fmul2(r, r), q, r);
  float2 s;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(n.x));      // a power of two
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(n.y));
  return ffma2(p, s, s);
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
  __device__ __forceinline__ void zero() { raw = make_uint4(0, 0, 0, 0); }
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
  __device__ __forceinline__ void zero() { raw = from_f32<T>(0.f); }
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
template <int VEC> __device__ __forceinline__ void store_f32(float* p, const float (&x)[VEC]) {
  if constexpr (VEC == 1) {
    *p = x[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  }
}
template <int VEC> __device__ __forceinline__ void decay(float (&a)[VEC]) {
  if constexpr (VEC == 1) {
    a[0] = decay2(make_float2(a[0], a[0])).x;
  } else {
#pragma unroll
    for (int i = 0; i < VEC; i += 2) {
      const float2 d = decay2(make_float2(a[i], a[i + 1]));
      a[i] = d.x; a[i + 1] = d.y;
    }
  }
}

// ---------------------------------------------------------------- composing runs

// Geometry of a block: CX threads side by side hold the channels of a token, kThreads / CX runs of R tokens lie below one
// another; a warp holds 32 / CX of them.
template <typename T, int VEC, int R_> struct Tile {
  static constexpr int CX = VEC == 1 ? 32 : 64 / VEC;
  static constexpr int C = CX * VEC;
  static constexpr int R = R_;
  static constexpr int kTokens = kThreads / CX * R;
};

// Runs composed over the lanes of a warp that hold the same channels, those of lower lanes first (or, with Reverse, last).
// On return (A, X) is the run of all lanes up to and with this one, (Ab, Xb) of those before it.
template <int VEC, int CX, bool Reverse>
__device__ __forceinline__ void compose_warp(float (&A)[VEC], float (&X)[VEC], float (&Ab)[VEC], float (&Xb)[VEC], int lane) {
#pragma unroll
  for (int off = CX; off < 32; off *= 2) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float a = Reverse ? __shfl_down_sync(0xffffffffu, A[i], off) : __shfl_up_sync(0xffffffffu, A[i], off);
      const float x = Reverse ? __shfl_down_sync(0xffffffffu, X[i], off) : __shfl_up_sync(0xffffffffu, X[i], off);
      if (Reverse ? lane + off < 32 : lane >= off) {
        X[i] = fmaf(A[i], x, X[i]);
        A[i] *= a;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    Ab[i] = 1.f;
    Xb[i] = 0.f;
    if constexpr (CX < 32) {
      const float a = Reverse ? __shfl_down_sync(0xffffffffu, A[i], CX) : __shfl_up_sync(0xffffffffu, A[i], CX);
      const float x = Reverse ? __shfl_down_sync(0xffffffffu, X[i], CX) : __shfl_up_sync(0xffffffffu, X[i], CX);
      if (Reverse ? lane + CX < 32 : lane >= CX) {
        Ab[i] = a;
        Xb[i] = x;
      }
    }
  }
}

// A warp's whole run per channel; the composing threads turn it into the run of the warps before.
template <int C> struct WarpRuns {
  float A[kWarps][C], X[kWarps][C];
};

// One thread per channel: the runs of the warps become those of the warps before each; (A, X) is the tile's run.
template <int C, bool Reverse>
__device__ __forceinline__ void compose_block(WarpRuns<C>& s, int c, float& A, float& X) {
  float a[kWarps], x[kWarps];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) { a[w] = s.A[w][c]; x[w] = s.X[w][c]; }
  A = 1.f;
  X = 0.f;
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    const int w = Reverse ? kWarps - 1 - i : i;
    s.A[w][c] = A;
    s.X[w][c] = X;
    X = fmaf(a[w], X, x[w]);
    A *= a[w];
  }
}

// ---------------------------------------------------------------- runs of the blocks of a cluster

template <int C> struct Exchange {                    // double buffered by the parity of the round
  float2 run[2][kMaxCluster][C];
  uint64_t bar[2];
  int abort;
};

__device__ __forceinline__ void send_run(uint32_t slot, uint32_t bar, int to, float A, float X) {
  uint32_t rslot, rbar;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rslot) : "r"(slot), "r"(to));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rbar) : "r"(bar), "r"(to));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];"
               ::"r"(rslot), "f"(A), "f"(X), "r"(rbar) : "memory");
}

// By the threads of the first C / 32 warps, one per channel: the run of this block's tile goes to every block of the cluster;
// returns what enters this tile and moves `carry` past the tiles of the whole cluster. Round `it` writes slots that the
// others read in round it - 2: nobody sends round it before its own round it - 1 is complete, which every block entered only
// after reading round it - 2.
template <int C>
__device__ __forceinline__ float enter_tile(Exchange<C>& ex, int it, int rank, int CL, int c, float A, float X, float& carry,
                                            uint32_t* status) {
  if (CL == 1) {
    const float in = carry;
    carry = fmaf(A, carry, X);
    return in;
  }
  const int p = it & 1;
  if (c == 0) tc::mbar_expect_tx(&ex.bar[p], (uint32_t)(CL * C * sizeof(float2)));
  const uint32_t slot = tc::smem_u32(&ex.run[p][rank][c]), bar = tc::smem_u32(&ex.bar[p]);
  for (int to = 0; to < CL; ++to) send_run(slot, bar, to, A, X);
  float in = carry;
  if (tc::mbar_wait_warp(&ex.bar[p], (it >> 1) & 1, &ex.abort, status, 1u << 29)) {
    for (int r = 0; r < CL; ++r) {
      if (r == rank) in = carry;
      const float2 run = ex.run[p][r][c];
      carry = fmaf(run.x, carry, run.y);
    }
  }
  return in;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <int C> __device__ __forceinline__ void init_exchange(Exchange<C>& ex, int CL, int tid) {
  if (tid == 0) {
    ex.abort = 0;
    tc::mbar_init(&ex.bar[0], 1);
    tc::mbar_init(&ex.bar[1], 1);
    tc::mbar_init_fence();
  }
  if (CL > 1) cluster_sync(); else __syncthreads();
}

struct Place {                     // a block's sequence, channel group and cluster
  int seq, group, rank, CL;
  int64_t start, len, mark;
};
template <bool Packed>
__device__ __forceinline__ Place place(const Args& a, const Tables& tb) {
  Place p;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(p.rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(p.CL));
  const int id = blockIdx.x / p.CL;
  p.group = id % a.groups;
  p.seq = id / a.groups;
  if constexpr (Packed) {
    p.start = tb.tok[p.seq];
    p.len = tb.tok[p.seq + 1] - p.start;
    p.mark = tb.mark[p.seq];
  } else {
    p.start = 0;
    p.len = a.S;
    p.mark = (int64_t)p.seq * ((a.S + kMarkTokens - 1) / kMarkTokens);
  }
  return p;
}

// ---------------------------------------------------------------- forward

template <typename T, int VEC, int R, bool Gate, bool Packed>
__global__ void __launch_bounds__(kThreads, 2) scan_forward_kernel(const __grid_constant__ Args a, const __grid_constant__ Tables tb,
                                                                   uint32_t* status) {
  using G = Tile<T, VEC, R>;
  constexpr int C = G::C, CX = G::CX;
  __shared__ WarpRuns<C> runs[2];
  __shared__ Exchange<C> ex;
  __shared__ float entering[2][C];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, cx = tid % CX, ry = tid / CX;
  const Place p = place<Packed>(a, tb);
  init_exchange(ex, p.CL, tid);

  const int c0 = p.group * C + cx * VEC;              // this thread's channels
  const bool live = c0 < a.D;
  const int64_t b = Packed ? 0 : p.seq, at = p.start;
  const T* v = static_cast<const T*>(a.v) + b * a.v_bs + at * a.v_ts + c0;
  const T* w = Gate ? static_cast<const T*>(a.w) + b * a.w_bs + at * a.w_ts + c0 : nullptr;
  const float* g = a.g + b * a.g_bs + at * a.g_ts + c0;
  T* o = static_cast<T*>(a.o) + (b * a.S + at) * a.D + c0;
  const int cc = p.group * C + tid;                   // the composing threads' channel
  float carry = 0.f;
  if (tid < C && cc < a.D && a.first) carry = a.first[(int64_t)p.seq * a.D + cc];

  const int64_t tiles = (p.len + G::kTokens - 1) / G::kTokens, rounds = (tiles + p.CL - 1) / p.CL;
  for (int64_t it = 0; it < rounds; ++it) {
    const int q = (int)(it & 1);
    const int64_t t0 = (it * p.CL + p.rank) * G::kTokens + ry * R;
    float dec[R][VEC], x[R][VEC];
    {
      Piece<T, VEC> pv[R], pw[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool in = live && t0 + r < p.len;
        pv[r].zero();
        if constexpr (Gate) pw[r].zero();
#pragma unroll
        for (int i = 0; i < VEC; ++i) dec[r][i] = 0.f;       // rows behind the end change nothing: decay 1, input 0
        if (in) {
          pv[r].load(v + (t0 + r) * a.v_ts);
          if constexpr (Gate) pw[r].load(w + (t0 + r) * a.w_ts);
          load_f32<VEC>(dec[r], g + (t0 + r) * a.g_ts);
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        decay<VEC>(dec[r]);
        pv[r].get(x[r]);
        if constexpr (Gate) {
          float wf[VEC];
          pw[r].get(wf);
#pragma unroll
          for (int i = 0; i < VEC; ++i) x[r][i] *= wf[i];
        }
      }
    }
    float A[VEC], X[VEC], Ab[VEC], Xb[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      A[i] = dec[0][i];
      X[i] = x[0][i];
#pragma unroll
      for (int r = 1; r < R; ++r) {
        X[i] = fmaf(dec[r][i], X[i], x[r][i]);
        A[i] *= dec[r][i];
      }
    }
    compose_warp<VEC, CX, false>(A, X, Ab, Xb, lane);
    if (lane >= 32 - CX) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) { runs[q].A[wid][cx * VEC + i] = A[i]; runs[q].X[wid][cx * VEC + i] = X[i]; }
    }
    __syncthreads();
    if (tid < C) {
      float At, Xt;
      compose_block<C, false>(runs[q], tid, At, Xt);
      entering[q][tid] = enter_tile<C>(ex, (int)it, p.rank, p.CL, tid, At, Xt, carry, status);
    }
    __syncthreads();
    float h[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const float in = fmaf(runs[q].A[wid][cx * VEC + i], entering[q][cx * VEC + i], runs[q].X[wid][cx * VEC + i]);
      h[i] = fmaf(Ab[i], in, Xb[i]);
    }
    if (a.marks && live && (ry * R) % kMarkTokens == 0 && t0 < p.len)
      store_f32<VEC>(a.marks + (p.mark + t0 / kMarkTokens) * a.D + c0, h);
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) h[i] = fmaf(dec[r][i], h[i], x[r][i]);
      if (live && t0 + r < p.len) Piece<T, VEC>::store(o + (t0 + r) * a.D, h);
    }
  }
  if (a.last && p.rank == 0 && tid < C && cc < a.D) a.last[(int64_t)p.seq * a.D + cc] = carry;
  if (p.CL > 1) cluster_sync();                       // no block leaves while another may still send to it
}

// ---------------------------------------------------------------- backward

// Tiles of 64 tokens, the last first: block `rank` of round `it` takes tile tiles - 1 - (it CL + rank).
template <typename T, int VEC, int R, bool Gate, bool Packed>
__global__ void __launch_bounds__(kThreads, 2) scan_backward_kernel(const __grid_constant__ Args a, const __grid_constant__ Tables tb,
                                                                    uint32_t* status) {
  using G = Tile<T, VEC, R>;
  static_assert(G::kTokens == kMarkTokens, "a tile starts at a mark");
  constexpr int C = G::C, CX = G::CX;
  __shared__ WarpRuns<C> runs[2], back[2];
  __shared__ Exchange<C> ex;
  __shared__ float entering[2][C], from_behind[2][C];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, cx = tid % CX, ry = tid / CX;
  const Place p = place<Packed>(a, tb);
  init_exchange(ex, p.CL, tid);

  const int c0 = p.group * C + cx * VEC;
  const bool live = c0 < a.D;
  const int64_t b = Packed ? 0 : p.seq, at = p.start;
  const T* v = static_cast<const T*>(a.v) + b * a.v_bs + at * a.v_ts + c0;
  const T* w = Gate ? static_cast<const T*>(a.w) + b * a.w_bs + at * a.w_ts + c0 : nullptr;
  const T* dout = static_cast<const T*>(a.dout) + b * a.do_bs + at * a.do_ts + c0;
  const float* g = a.g + b * a.g_bs + at * a.g_ts + c0;
  const int64_t out0 = (b * a.S + at) * a.D + c0;
  const int cc = p.group * C + tid;
  float carry = 0.f;
  if (tid < C && cc < a.D && a.first) carry = a.first[(int64_t)p.seq * a.D + cc];

  const int64_t tiles = (p.len + G::kTokens - 1) / G::kTokens, rounds = (tiles + p.CL - 1) / p.CL;
  for (int64_t it = 0; it < rounds; ++it) {
    const int q = (int)(it & 1);
    const int64_t tile = tiles - 1 - (it * p.CL + p.rank), t0 = tile * G::kTokens + ry * R;
    Piece<T, VEC> pv[R], pw[R], pd[R];
    float dec[R][VEC];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool in = live && t0 + r >= 0 && t0 + r < p.len;
      pv[r].zero();
      pd[r].zero();
      if constexpr (Gate) pw[r].zero();
#pragma unroll
      for (int i = 0; i < VEC; ++i) dec[r][i] = 0.f;
      if (in) {
        pv[r].load(v + (t0 + r) * a.v_ts);
        pd[r].load(dout + (t0 + r) * a.do_ts);
        if constexpr (Gate) pw[r].load(w + (t0 + r) * a.w_ts);
        load_f32<VEC>(dec[r], g + (t0 + r) * a.g_ts);
      }
    }
    // C + tid threads compose the forward runs from the tile's mark, tid threads the backward ones
    if (tid >= C && tid < 2 * C) {
      const int c = p.group * C + tid - C;
      entering[q][tid - C] = tile >= 0 && c < a.D ? a.marks[(p.mark + tile) * a.D + c] : 0.f;
    }
    float A[VEC], X[VEC], Ab[VEC], Xb[VEC], Br[VEC], Y[VEC], Bb[VEC], Yb[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) { A[i] = 1.f; X[i] = 0.f; Y[i] = 0.f; }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      decay<VEC>(dec[r]);
      float vf[VEC], wf[VEC];
      pv[r].get(vf);
      if constexpr (Gate) pw[r].get(wf);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float x = Gate ? vf[i] * wf[i] : vf[i];
        X[i] = fmaf(dec[r][i], X[i], x);
        A[i] *= dec[r][i];
      }
    }
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      float df[VEC];
      pd[r].get(df);
#pragma unroll
      for (int i = 0; i < VEC; ++i) Y[i] = dec[r][i] * (df[i] + Y[i]);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) Br[i] = A[i];
    compose_warp<VEC, CX, false>(A, X, Ab, Xb, lane);
    compose_warp<VEC, CX, true>(Br, Y, Bb, Yb, lane);
    if (lane >= 32 - CX) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) { runs[q].A[wid][cx * VEC + i] = A[i]; runs[q].X[wid][cx * VEC + i] = X[i]; }
    }
    if (lane < CX) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) { back[q].A[wid][cx * VEC + i] = Br[i]; back[q].X[wid][cx * VEC + i] = Y[i]; }
    }
    __syncthreads();
    if (tid < C) {
      float At, Yt;
      compose_block<C, true>(back[q], tid, At, Yt);
      from_behind[q][tid] = enter_tile<C>(ex, (int)it, p.rank, p.CL, tid, At, Yt, carry, status);
    } else if (tid < 2 * C) {
      float At, Xt;
      compose_block<C, false>(runs[q], tid - C, At, Xt);
    }
    __syncthreads();
    float before[R][VEC], h[VEC], cf[VEC];             // before: a_t h_{t-1}
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int c = cx * VEC + i;
      h[i] = fmaf(Ab[i], fmaf(runs[q].A[wid][c], entering[q][c], runs[q].X[wid][c]), Xb[i]);
      cf[i] = fmaf(Bb[i], fmaf(back[q].A[wid][c], from_behind[q][c], back[q].X[wid][c]), Yb[i]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float vf[VEC], wf[VEC];
      pv[r].get(vf);
      if constexpr (Gate) pw[r].get(wf);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float x = Gate ? vf[i] * wf[i] : vf[i];
        before[r][i] = h[i];
        h[i] = fmaf(dec[r][i], h[i], x);
      }
    }
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      const bool in = live && t0 + r >= 0 && t0 + r < p.len;
      float vf[VEC], wf[VEC], df[VEC], dv[VEC], dw[VEC], dg[VEC];
      pd[r].get(df);
      pv[r].get(vf);
      if constexpr (Gate) pw[r].get(wf);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float dh = df[i] + cf[i];
        dv[i] = Gate ? dh * wf[i] : dh;
        dw[i] = dh * vf[i];
        cf[i] = dec[r][i] * dh;
        dg[i] = cf[i] * before[r][i];
      }
      if (in) {
        const int64_t e = out0 + (t0 + r) * a.D;
        Piece<T, VEC>::store(static_cast<T*>(a.dv) + e, dv);
        if constexpr (Gate) Piece<T, VEC>::store(static_cast<T*>(a.dw) + e, dw);
        store_f32<VEC>(a.dg + e, dg);
      }
    }
  }
  if (a.last && p.rank == 0 && tid < C && cc < a.D) a.last[(int64_t)p.seq * a.D + cc] = carry;
  if (p.CL > 1) cluster_sync();
}

// ---------------------------------------------------------------- few tokens

// At most kStepTokens tokens: a thread takes its channels of a sequence through all of them. The state may be updated in place.
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
  if (a.first) load_f32<VEC>(h, a.first + seq * a.D + c0);
  const int S = (int)a.S;
  for (int t = 0; t < S; ++t) {
    Piece<T, VEC> pv, pw;
    float dec[VEC], x[VEC], wf[VEC];
    pv.load(v + t * a.v_ts);
    if constexpr (Gate) pw.load(w + t * a.w_ts);
    load_f32<VEC>(dec, g + t * a.g_ts);
    decay<VEC>(dec);
    pv.get(x);
    if constexpr (Gate) pw.get(wf);
#pragma unroll
    for (int i = 0; i < VEC; ++i) h[i] = fmaf(dec[i], h[i], Gate ? x[i] * wf[i] : x[i]);
    Piece<T, VEC>::store(o + (int64_t)t * a.D, h);
  }
  if (a.last) store_f32<VEC>(a.last + seq * a.D + c0, h);
}

// ---------------------------------------------------------------- launches

// Blocks per cluster: 2 blocks fit on an SM, so the tiles of a sequence are spread over as many blocks as it takes to fill the
// GPU so, as long as there are tiles for them.
int cluster_size(int64_t sequences, int groups, int64_t tiles) {
  const int64_t want = 2 * device_sm_count();
  int cl = 1;
  while (cl < kMaxCluster && sequences * groups * cl < want && 2 * cl <= tiles) cl *= 2;
  return cl;
}

template <typename... P>
int launch_clustered(void (*kernel)(P...), int64_t clusters, int cl, cudaStream_t st, const Args& a, const Tables& tb) {
  uint32_t* status = device_status_word();
  if (!status) return record_cuda_error(cudaGetLastError());
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cl;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(clusters * cl));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  GDN2_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, tb, status));
  return GDN2_OK;
}

template <typename T, int VEC, bool Gate, bool Packed>
int launch_scan(const Args& a0, const Tables& tb, int64_t longest, bool backward, cudaStream_t st) {
  constexpr int RF = VEC == 1 ? 8 : 32 / VEC, RB = VEC == 1 ? 8 : 16 / VEC;
  using F = Tile<T, VEC, RF>;
  Args a = a0;
  a.groups = (a.D + F::C - 1) / F::C;
  const int tile = backward ? kMarkTokens : F::kTokens;
  const int64_t clusters = (int64_t)a.sequences * a.groups;
  const int cl = cluster_size(a.sequences, a.groups, (longest + tile - 1) / tile);
  if (clusters * cl > 2147483647LL) return GDN2_ERR_BAD_SHAPE;
  if (backward) return launch_clustered(scan_backward_kernel<T, VEC, RB, Gate, Packed>, clusters, cl, st, a, tb);
  return launch_clustered(scan_forward_kernel<T, VEC, RF, Gate, Packed>, clusters, cl, st, a, tb);
}

template <typename T, int VEC, bool Gate>
int launch_all(const Args& a, const int64_t* cu, bool backward, cudaStream_t st) {
  if (!cu) {
    Tables none;
    none.n = 0;
    if (!backward && a.S <= kStepTokens && !a.marks) {
      const int64_t threads = (int64_t)a.sequences * ((a.D + VEC - 1) / VEC), blocks = (threads + 127) / 128;
      if (blocks > 2147483647LL) return GDN2_ERR_BAD_SHAPE;
      scan_steps_kernel<T, VEC, Gate><<<(unsigned)blocks, 128, 0, st>>>(a);
      GDN2_CUDA_TRY(cudaGetLastError());
      return GDN2_OK;
    }
    return launch_scan<T, VEC, Gate, false>(a, none, a.S, backward, st);
  }
  int64_t mark = 0;
  for (int i0 = 0; i0 < a.sequences; i0 += kMaxPacked) {
    Tables tb;
    tb.n = a.sequences - i0 < kMaxPacked ? a.sequences - i0 : kMaxPacked;
    int64_t longest = 0;
    for (int i = 0; i <= tb.n; ++i) {
      tb.tok[i] = (int)cu[i0 + i];
      tb.mark[i] = (int)mark;
      if (i < tb.n) {
        const int64_t len = cu[i0 + i + 1] - cu[i0 + i];
        longest = len > longest ? len : longest;
        mark += (len + kMarkTokens - 1) / kMarkTokens;
      }
    }
    Args part = a;
    part.sequences = tb.n;
    if (a.first) part.first = a.first + (int64_t)i0 * a.D;
    if (a.last) part.last = a.last + (int64_t)i0 * a.D;
    const int rc = launch_scan<T, VEC, Gate, true>(part, tb, longest, backward, st);
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

// 16-byte pieces need rows that start on 16 bytes and a number of channels that pieces divide
bool all_wide(const gdn2_recurrence_args& r, int dtype, bool backward) {
  const int64_t esz = dtype == GDN2_F32 ? 4 : 2, V = 16 / esz;
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  auto rows = [&](const void* p, int64_t bs, int64_t ts, int64_t size) {
    return !p || (aligned(p) && bs * size % 16 == 0 && ts * size % 16 == 0);
  };
  if (r.D % V) return false;
  if (!rows(r.v, r.v_batch_stride, r.v_token_stride, esz) || !rows(r.g, r.g_batch_stride, r.g_token_stride, 4) ||
      !rows(r.w, r.w_batch_stride, r.w_token_stride, esz) || !aligned(r.state) || !aligned(r.final_state) || !aligned(r.marks))
    return false;
  if (!backward) return aligned(r.o);
  return rows(r.dout, r.do_batch_stride, r.do_token_stride, esz) && aligned(r.dv) && aligned(r.dw) && aligned(r.dg);
}

int run(const gdn2_recurrence_args& r, int dtype, bool backward, cudaStream_t st) {
  const int rc = check(r, dtype, backward);
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
  const int64_t m = gdn2::kMarkTokens;
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
