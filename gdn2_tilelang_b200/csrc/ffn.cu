// The gated feed-forward block y = (act(x Wg^T) * (x Wu^T)) Wd^T and its gradient, 16-bit operands, fp32 accumulation.
//
//   forward   a = x Wg^T, u = x Wu^T, h = act(a) u     one kernel: both projections, the activation and the product
//             y = h Wd^T
//   backward  dh = dy Wd, da = dh u act'(a), du = dh act(a), h again      one kernel
//             dx = da Wg + du Wu                                 one kernel (the two products are one long reduction)
//             dWg = da^T x, dWu = du^T x;  dWd = dy^T h          a kernel each
//
// Every product is the same pipeline with another way in and another way out (product_kernel): a pair of blocks on two SMs
// (cta_group::2) holds a 256 x 256 tile of the result in tensor memory, 128 rows each; TMA brings 64 reduction steps of both
// operands a stage, each block its own 128 rows of A and its half of B's, six stages deep (four where gradients need the room); one thread issues the products;
// eight warps take the finished tile from tensor memory while the next one accumulates in the other half of it. The operands are read
// as they lie in memory: with the reduction along rows (K-major) or down columns (MN-major), which the shared-memory
// descriptors tell the tensor core, so nothing is transposed.
//
// In the forward product block 0 of a pair brings rows of Wg as its half of B and block 1 the same rows of Wu: columns c and 128 + c of
// the tile are then the gate and the up projection of one inner channel, in the same lane of tensor memory, and the epilogue
// needs nothing from another thread. h is rounded to 16 bits there: it is what the next product reads, and a tensor core reads
// 16 bits. The same holds for da and du. Everything else stays fp32 up to the results, with one exception: what a training step
// keeps of a and u are the upper 24 bits of their fp32 sums, 16 in one plane and 8 in another. In 16 bits their rounding weighs as
// much as that of da or of the result (dx off by 3.1e-3 of its 2-norm in bf16, with 24 bits by 2.4e-3); keeping them so and forming h a second
// time in the backward pass takes the 6 bytes an inner channel that a, u and h take in 16 bits.
//
// Few tokens (skinny_kernel): the work is reading the weights once. They take the 128-row side of the product, the tokens
// the narrow one, and the reduction of a tile is cut over the blocks of a cluster so that every SM reads; the blocks' partial
// sums meet in distributed shared memory, added in the order of the blocks. The second kernel is chained to the first: it asks for its
// first weights, which nothing before it writes, as soon as it finds a place, and for the first's results when that has completed.
// The first is launched plainly, so everything before it is complete by then.
#include "clusters.cuh"
#include "common.cuh"
#include "tc_utils.cuh"
#include "tensor_map.cuh"

namespace gdn2 {

namespace {

constexpr int kTile = 256;                       // rows and columns of a pair's tile
constexpr int kBlockRows = 128, kStep = 64;      // a block's rows of an operand, reduction steps of a stage
constexpr int kOperandBytes = kBlockRows * kStep * 2;
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kEpiWarps = 8, kThreads = (4 + kEpiWarps) * 32;
constexpr int kChunk16 = 64;                     // columns of an epilogue chunk: 128 bytes
constexpr int kChunkBytes = 32 * kChunk16 * 2;
constexpr uint32_t kWaitCode = 1u << 28;

enum Kind { kPlain = 0, kGated = 1, kGatedBackward = 2 };

// Stages that fit beside a kind's staging buffers: one chunk a warp; for the backward epilogue 6 KB in and 6 KB out.
template <int K> __host__ __device__ constexpr int stages() { return K == kGatedBackward ? 4 : 6; }
template <int K> __host__ __device__ constexpr int staging_bytes() { return kEpiWarps * kChunkBytes * (K == kGatedBackward ? 3 : 1); }
template <int K> constexpr size_t smem_bytes() { return (size_t)stages<K>() * kStageBytes + staging_bytes<K>() + 1024; }

struct __align__(64) Maps {
  CUtensorMap a[2], b[2];       // kPlain: operands of the one or two runs of reduction steps; kGated: b = Wg, Wu
  CUtensorMap out[3];           // kPlain: result (of the upper and of the lower tiles); kGated: h; kGatedBackward: da, du, h
  CUtensorMap kept[4];          // the planes of a and u: upper 16 bits of a, of u, lower 8 of a, of u
};
struct Problem {
  int steps[2];                 // stages of the two runs (steps[1] = 0: one run)
  int tiles_m, tiles_n;
  int split_m;                  // > 0: tiles from this one on take a[1] and out[1], their rows counted from there (dWg, dWu)
  int M, N;                     // rows and columns of the result (of one part)
  int split;                    // kPlain: pairs of a cluster that share a tile's reduction; > 1: a cluster a tile
  int save;                     // kGated: a and u are kept; kGatedBackward: h is wanted
  void* plain_out[2];           // results whose rows do not start on 16 bytes are stored by threads
  int64_t out_stride;
};

// The planes of a and u inside a kept buffer of 6 tokens * stride bytes
struct Planes {
  uint16_t* upper[2];
  uint8_t* lower[2];
};
__host__ __device__ inline Planes planes(void* kept, int64_t tokens, int64_t stride) {
  const int64_t n = tokens * stride;
  Planes p;
  p.upper[0] = static_cast<uint16_t*>(kept);
  p.upper[1] = p.upper[0] + n;
  p.lower[0] = reinterpret_cast<uint8_t*>(p.upper[1] + n);
  p.lower[1] = p.lower[0] + n;
  return p;
}

// ---------------------------------------------------------------- instructions

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t in_block(uint32_t addr, uint32_t rank) {       // the same shared address in another block
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
               ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, int x, int y, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];"
               ::"l"(map), "r"(x), "r"(y), "r"(src) : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// arrives on the barrier at this offset of both blocks of a pair once every product issued so far has completed
__device__ __forceinline__ void commit_pair(uint64_t* bar, uint32_t leader) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(tc::smem_u32(bar)), "h"((uint16_t)(3u << leader)) : "memory");
}
// A lane has read what it will of the memory that this barrier stands for: the arrival comes after its loads
__device__ __forceinline__ void arrive_read(uint64_t* bar) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(tc::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Descriptor of a 128-byte-swizzled operand tile as TMA writes it.
//   K-major:  rows of 64 reduction steps (128 bytes), 1024 bytes from one group of 8 rows to the next; 16 steps are 32 bytes.
//   MN-major: a piece is 64 rows of A (or B) wide and 64 steps tall, 128 bytes a step; 1024 bytes from 8 steps to the next 8,
//             8192 from one piece to the next; 16 steps are 2048 bytes.
template <bool MN> __device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  uint64_t d = (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)((MN ? 8192u : 16u) >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= 1ull << 46;
  d |= 2ull << 61;
  return d;
}
template <bool MN> __host__ __device__ constexpr uint32_t operand_step() { return (MN ? 2048u : 32u) >> 4; }

template <typename T> struct Format { static constexpr uint32_t code = 0; };                       // fp16
template <> struct Format<__nv_bfloat16> { static constexpr uint32_t code = 1; };
template <typename T> __host__ __device__ constexpr uint32_t idesc_of(bool a_mn, bool b_mn, uint32_t M, uint32_t N) {
  return tc::instr_desc(Format<T>::code, M, N) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
}

// ---------------------------------------------------------------- activation

// act(a) and, where wanted, act'(a). Both are a times a logistic function: silu s(a), gelu's tanh form s(2 z) with
// z = sqrt(2 / pi) (a + 0.044715 a^3). Beyond |a| = 16 the latter is 0 or 1 to 32 bits; z stops there so that a^3 stays finite
// (by a clamp that leaves a NaN one: a slope of 0 in its place would keep it out of the gate's gradient).
// (A template argument: with a branch on it inside the epilogue's loops the backward one took 250 us instead of 209, 8192 x 2048 x 5632.)
// The exponential and the reciprocal are the approximate instructions: 2^-21, against results of 11 bits at most.
__device__ __forceinline__ float clamp_or_nan(float x, float most) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(-most));
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(r), "f"(most));
  return r;
}
__device__ __forceinline__ float logistic(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
template <bool Gelu, bool Slope> __device__ __forceinline__ float activate(float a, float& slope) {
  if constexpr (Gelu) {
    const float c = 0.7978845608028654f, t = clamp_or_nan(a, 16.f), t2 = t * t;
    const float s = logistic(2.f * c * t * fmaf(0.044715f, t2, 1.f));
    if constexpr (Slope) slope = fmaf(2.f * c * t * s * (1.f - s), fmaf(3.f * 0.044715f, t2, 1.f), s);
    return a * s;
  } else {
    const float s = logistic(a);
    if constexpr (Slope) slope = s * fmaf(a, 1.f - s, 1.f);
    return a * s;
  }
}

// ---------------------------------------------------------------- the epilogue's chunks: 32 rows of 64 columns, swizzled

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 t = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&t);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&t);
}
// 32 columns from `first` (0 or 32) of this lane's row
template <typename T> __device__ __forceinline__ void put_row(char* chunk, int lane, int first, const float (&x)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4 r;
    r.x = pack2<T>(x[8 * j], x[8 * j + 1]); r.y = pack2<T>(x[8 * j + 2], x[8 * j + 3]);
    r.z = pack2<T>(x[8 * j + 4], x[8 * j + 5]); r.w = pack2<T>(x[8 * j + 6], x[8 * j + 7]);
    *reinterpret_cast<uint4*>(chunk + lane * 128 + (((first / 8 + j) ^ (lane & 7)) * 16)) = r;
  }
}
// The upper 24 bits of two or four numbers, rounded (ties away from zero; a number within 2^-17 of the largest becomes infinite).
// A NaN keeps its upper 16 bits, whose quiet bit is set.
__device__ __forceinline__ uint32_t round24(float x) {
  const uint32_t b = __float_as_uint(x);
  return (b & 0x7fffffffu) > 0x7f800000u ? b : b + 0x80u;
}
__device__ __forceinline__ uint32_t upper16(uint32_t b0, uint32_t b1) { return __byte_perm(b0, b1, 0x7632); }
__device__ __forceinline__ uint32_t lower8(uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
  return __byte_perm(__byte_perm(b0, b1, 0x0051), __byte_perm(b2, b3, 0x0051), 0x5410);
}
// 32 columns from `first` (0 or 32) of this lane's row of the upper plane's chunk, from rounded numbers
__device__ __forceinline__ void put_upper(char* chunk, int lane, int first, const uint32_t (&b)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(chunk + lane * 128 + (((first / 8 + j) ^ (lane & 7)) * 16)) =
        make_uint4(upper16(b[8 * j], b[8 * j + 1]), upper16(b[8 * j + 2], b[8 * j + 3]), upper16(b[8 * j + 4], b[8 * j + 5]),
                   upper16(b[8 * j + 6], b[8 * j + 7]));
}
// Rows of 64 bytes, swizzled as TMA does it: of the forward chunk's lower planes, and of the backward epilogue's pieces, which are 32
// columns (their lower planes have rows of 32 bytes).
__device__ __forceinline__ uint32_t row64_at(int lane, int j) { return lane * 64 + ((j ^ ((lane >> 1) & 3)) * 16); }
template <typename T> __device__ __forceinline__ void put_row64(char* piece, int lane, const float (&x)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint4 r;
    r.x = pack2<T>(x[8 * j], x[8 * j + 1]); r.y = pack2<T>(x[8 * j + 2], x[8 * j + 3]);
    r.z = pack2<T>(x[8 * j + 4], x[8 * j + 5]); r.w = pack2<T>(x[8 * j + 6], x[8 * j + 7]);
    *reinterpret_cast<uint4*>(piece + row64_at(lane, j)) = r;
  }
}
__device__ __forceinline__ void get_kept(const char* upper, const char* lower, int lane, float (&x)[32]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint4 lo = *reinterpret_cast<const uint4*>(lower + lane * 32 + ((half ^ ((lane >> 2) & 1)) * 16));
    const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint4 r = *reinterpret_cast<const uint4*>(upper + row64_at(lane, 2 * half + j));
      const uint32_t h[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int i = 0; i < 8; ++i)     // two bytes of the upper plane, one of the lower
        x[16 * half + 8 * j + i] =
            __uint_as_float(__byte_perm(h[i / 2], l[2 * j + i / 4], (i & 1 ? 0x3200 : 0x1000) | (4 + (i & 3)) << 4) & 0xffffff00u);
    }
  }
}
// A warp's chunk to rows row.., columns col.. of the result; what lies outside is dropped.
template <typename T>
__device__ __forceinline__ void store_chunk(const char* chunk, const CUtensorMap* map, T* plain, int64_t stride, int row, int col, int M,
                                            int N, int lane) {
  if (row >= M || col >= N) return;
  if (plain == nullptr) {
    tc::fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      tma_store(map, col, row, tc::smem_u32(chunk));
      tc::bulk_commit();
    }
    return;
  }
  __syncwarp();
  for (int r = 0; r < 32 && row + r < M; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = lane + 32 * h;
      const T e = *reinterpret_cast<const T*>(chunk + r * 128 + (((c >> 3) ^ (r & 7)) * 16) + (c & 7) * 2);
      if (col + c < N) plain[(int64_t)(row + r) * stride + col + c] = e;
    }
}
__device__ __forceinline__ void chunk_free(int lane) {        // the chunk may be written again
  if (lane == 0) tc::bulk_wait_read_all();
  __syncwarp();
}

// ---------------------------------------------------------------- tiles of 256 x 256

struct Shared {
  uint64_t full[8], empty[8], done[2], taken[2], loaded[kEpiWarps], read[kEpiWarps];
  uint32_t tmem;
  int abort;
};

// Tiles go in bands of 16 rows of tiles, down the rows first, so that the pairs at work at one time share operands in L2.
__device__ __forceinline__ void tile_at(const Problem& p, int i, int& m, int& n) {
  const int band = 16, per = band * p.tiles_n, b = i / per, rows = min(band, p.tiles_m - b * band);
  m = b * band + (i - b * per) % rows;
  n = (i - b * per) / rows;
}

// The pairs of a cluster have each summed a part of one tile's reduction: each finishes 256 / split of its columns. What it has of the
// others' columns goes to their shared memory (the ring: every product has read it, in every block of the cluster), and the
// parts are added in their order. By all threads of all blocks of the cluster.
template <typename T>
__device__ __forceinline__ void join_parts(const Maps& maps, const Problem& p, Shared& sh, char* ring, char* staging, uint32_t tmem, int tile,
                                           int rank, int part, int split, uint32_t* status) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, quad = wid & 3, half = (wid - 4) >> 2;
  const int own = kTile / split, mine = own / 2;         // a pair's columns, a warp's
  bool ok = false;
  if (wid >= 4) {
    ok = tc::mbar_wait_warp(&sh.done[0], 0, &sh.abort, status, kWaitCode);
    tc::tc_fence_after_sync();
  }
  __syncthreads();
  cluster_sync();
  const uint32_t acc = tmem + ((uint32_t)(quad * 32) << 16);
  const uint32_t parts = tc::smem_u32(ring) + (quad * 32 + lane) * 16;      // [part][column / 4][row][4]
  if (ok)
    for (int o = 0; o < split; ++o) {
      if (o == part) continue;
      const uint32_t to = in_block(parts + (part < o ? part : part - 1) * own * kBlockRows * 4, 2 * o + rank);
      for (int c = half * mine; c < (half + 1) * mine; c += 32) {
        float x[32];
        tc::tmem_ld32(acc + o * own + c, x);
        tc::tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + (c / 4 + j) * kBlockRows * 16), "f"(x[4 * j]),
                       "f"(x[4 * j + 1]), "f"(x[4 * j + 2]), "f"(x[4 * j + 3]) : "memory");
      }
    }
  __syncthreads();
  cluster_sync();
  if (ok) {
    int m, n;
    tile_at(p, tile, m, n);
    const bool lower = p.split_m > 0 && m >= p.split_m;
    const int row = (lower ? m - p.split_m : m) * kTile + rank * kBlockRows + quad * 32;
    char* piece = staging + (wid - 4) * kChunkBytes;
    T* plain = static_cast<T*>(p.plain_out[lower]);
    for (int c = half * mine; c < (half + 1) * mine; c += 32) {
      float x[32], sum[32] = {};
      tc::tmem_ld32(acc + part * own + c, x);
      tc::tmem_ld_wait();
      for (int q = 0; q < split; ++q) {
        const uint32_t from = parts + (q < part ? q : q - 1) * own * kBlockRows * 4;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float4 f = make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
          if (q != part)
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w)
                         : "r"(from + (c / 4 + j) * kBlockRows * 16) : "memory");
          sum[4 * j] += f.x; sum[4 * j + 1] += f.y; sum[4 * j + 2] += f.z; sum[4 * j + 3] += f.w;
        }
      }
      const int col = n * kTile + part * own + c;
      chunk_free(lane);
      put_row64<T>(piece, lane, sum);
      if (row >= p.M || col >= p.N) continue;
      if (plain == nullptr) {
        tc::fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store(&maps.out[lower], col, row, tc::smem_u32(piece));
          tc::bulk_commit();
        }
      } else {
        __syncwarp();
        for (int r = 0; r < 32 && row + r < p.M; ++r)
          if (col + lane < p.N)
            plain[(int64_t)(row + r) * p.out_stride + col + lane] = *reinterpret_cast<const T*>(piece + row64_at(r, lane >> 3) + (lane & 7) * 2);
        __syncwarp();
      }
    }
    if (lane == 0) tc::bulk_wait_all();
    __syncwarp();
  }
  tc::tc_fence_before_sync();
}

template <typename T, int K, bool A_MN, bool B_MN, bool Gelu>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Problem p, uint32_t* status) {
  constexpr int S = stages<K>();
  extern __shared__ __align__(1024) char smem_raw[];
  __shared__ Shared sh;
  char* ring = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  char* staging = ring + S * kStageBytes;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const uint32_t block = cluster_rank(), rank = block & 1, leader = block & ~1u;
  const int split = K == kPlain ? p.split : 1, part = (int)block >> 1;      // pairs of the cluster, and which this is
  const int pair = blockIdx.x / (2 * split), pairs = gridDim.x / (2 * split);
  const int tiles = p.tiles_m * p.tiles_n, steps = p.steps[0] + p.steps[1];
  const int first = steps * part / split, behind = steps * (part + 1) / split;      // this pair's share of the reduction

  if (wid == 0 && lane == 0) {
    for (int i = 0; i < S; ++i) {
      tc::mbar_init(&sh.full[i], 1);
      tc::mbar_init(&sh.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&sh.done[i], 1);
      tc::mbar_init(&sh.taken[i], 2 * kEpiWarps);
    }
    for (int i = 0; i < kEpiWarps; ++i) {
      tc::mbar_init(&sh.loaded[i], 1);
      tc::mbar_init(&sh.read[i], 32);
    }
    sh.abort = 0;
    tc::mbar_init_fence();
  }
  if (wid == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(&sh.tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc::tc_fence_before_sync();
  __syncthreads();
  cluster_sync();
  tc::tc_fence_after_sync();
  const uint32_t tmem = sh.tmem;

  if (wid == 0) {
    // ---- copies: this block's rows of A and its half of B, counted on block 0's barrier
    if (lane == 0) {
      int s = 0, phase = 0;
      bool ok = true;
      for (int i = pair; ok && i < tiles; i += pairs) {
        int m, n;
        tile_at(p, i, m, n);
        const bool lower = p.split_m > 0 && m >= p.split_m;
        const int row_a = (lower ? m - p.split_m : m) * kTile + rank * kBlockRows;
        const int row_b = K == kGated ? n * kBlockRows : n * kTile + (int)rank * kBlockRows;
        for (int k = first; k < behind; ++k) {
          const int run = k >= p.steps[0], at = (run ? k - p.steps[0] : k) * kStep;
          const CUtensorMap* ma = &maps.a[lower || run ? 1 : 0];
          const CUtensorMap* mb = &maps.b[K == kGated ? (int)rank : run];
          if (!tc::mbar_wait(&sh.empty[s], phase ^ 1, &sh.abort, status, kWaitCode)) { ok = false; break; }
          const uint32_t bar = in_block(tc::smem_u32(&sh.full[s]), leader), dst = tc::smem_u32(ring + s * kStageBytes);
          if (rank == 0) tc::mbar_expect_tx(&sh.full[s], 2 * kStageBytes);
          if constexpr (A_MN) {
            tma_load_pair(dst, ma, row_a, at, bar);
            tma_load_pair(dst + kOperandBytes / 2, ma, row_a + 64, at, bar);
          } else {
            tma_load_pair(dst, ma, at, row_a, bar);
          }
          if constexpr (B_MN) {
            tma_load_pair(dst + kOperandBytes, mb, row_b, at, bar);
            tma_load_pair(dst + kOperandBytes + kOperandBytes / 2, mb, row_b + 64, at, bar);
          } else {
            tma_load_pair(dst + kOperandBytes, mb, at, row_b, bar);
          }
          if (++s == S) { s = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (wid == 1) {
    // ---- products: one thread of block 0 for both
    if (rank == 0 && lane == 0) {
      constexpr uint32_t idesc = idesc_of<T>(A_MN, B_MN, kTile, kTile);
      int s = 0, phase = 0, buf = 0, taken = 1;
      bool ok = true;
      for (int i = pair; ok && i < tiles; i += pairs) {
        if (!tc::mbar_wait(&sh.taken[buf], taken, &sh.abort, status, kWaitCode)) break;
        tc::tc_fence_after_sync();
        const uint32_t d = tmem + buf * kTile;
        for (int k = first; k < behind; ++k) {
          if (!tc::mbar_wait(&sh.full[s], phase, &sh.abort, status, kWaitCode)) { ok = false; break; }
          tc::tc_fence_after_sync();
          const uint32_t at = tc::smem_u32(ring + s * kStageBytes);
          uint64_t a = operand_desc<A_MN>(at), b = operand_desc<B_MN>(at + kOperandBytes);
#pragma unroll
          for (int q = 0; q < kStep / 16; ++q)
            mma_pair(d, a + q * operand_step<A_MN>(), b + q * operand_step<B_MN>(), idesc, k > first || q > 0);
          commit_pair(&sh.empty[s], leader);
          if (++s == S) { s = 0; phase ^= 1; }
        }
        if (ok) commit_pair(&sh.done[buf], leader);
        if (buf == 1) taken ^= 1;
        buf ^= 1;
      }
    }
    __syncwarp();
  } else if (wid >= 4) {
    // ---- results: lanes 32 (wid % 4).. of tensor memory, the first or the second half of the columns
    const int quad = wid & 3, half = (wid - 4) >> 2, ew = wid - 4;
    char* chunk = staging + ew * (staging_bytes<K>() / kEpiWarps);
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;
    const uint32_t taken0 = in_block(tc::smem_u32(&sh.taken[0]), leader), taken1 = in_block(tc::smem_u32(&sh.taken[1]), leader);
    int buf = 0, phase = 0;
    int loads = 0;                                    // kGatedBackward: pieces loaded so far
    auto load_piece = [&](int i, int c) {             // 32 columns of a and u, piece c of this warp's half of tile i
      if (i >= tiles) return;
      int m, n;
      tile_at(p, i, m, n);
      if (lane == 0) {
        const int row = m * kTile + rank * kBlockRows + quad * 32, col = n * kTile + half * 128 + c * 32;
        const uint32_t bar = tc::smem_u32(&sh.loaded[ew]), at = tc::smem_u32(chunk);
        tc::mbar_expect_tx(&sh.loaded[ew], 6144);
        tma_load(at, &maps.kept[0], col, row, bar);
        tma_load(at + 2048, &maps.kept[1], col, row, bar);
        tma_load(at + 4096, &maps.kept[2], col, row, bar);
        tma_load(at + 5120, &maps.kept[3], col, row, bar);
      }
    };
    if constexpr (K == kGatedBackward) load_piece(pair, 0);
    for (int i = pair; split == 1 && i < tiles; i += pairs) {
      int m, n;
      tile_at(p, i, m, n);
      const bool lower = p.split_m > 0 && m >= p.split_m;
      const int row = (lower ? m - p.split_m : m) * kTile + rank * kBlockRows + quad * 32;
      if (!tc::mbar_wait_warp(&sh.done[buf], phase, &sh.abort, status, kWaitCode)) break;
      tc::tc_fence_after_sync();
      const uint32_t acc = tmem + lanes + buf * kTile;
      if constexpr (K == kPlain) {
        const CUtensorMap* map = &maps.out[lower];
        T* plain = static_cast<T*>(p.plain_out[lower]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int at = half * 128 + c * kChunk16;
          float x[32];
          chunk_free(lane);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            tc::tmem_ld32(acc + at + 32 * q, x);
            tc::tmem_ld_wait();
            put_row<T>(chunk, lane, 32 * q, x);
          }
          store_chunk<T>(chunk, map, plain, p.out_stride, row, n * kTile + at, p.M, p.N, lane);
          if (plain) __syncwarp();
        }
      } else if constexpr (K == kGated) {
        const int col = n * kBlockRows + half * kChunk16;
        uint32_t alow[16], ulow[16];                  // the lower planes
#pragma unroll
        for (int part = 0; part < 3; ++part) {        // h, then the upper planes; the tile is read again for each rather than held
          if (part > 0 && !p.save) break;
          chunk_free(lane);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float a[32], u[32];
            if (part != 2) tc::tmem_ld32(acc + half * kChunk16 + 32 * q, a);
            if (part != 1) tc::tmem_ld32(acc + kBlockRows + half * kChunk16 + 32 * q, u);
            tc::tmem_ld_wait();
            if (part == 0) {
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                float none;
                a[j] = activate<Gelu, false>(a[j], none) * u[j];
              }
              put_row<T>(chunk, lane, 32 * q, a);
            } else {
              uint32_t b[32], (&low)[16] = part == 1 ? alow : ulow;
#pragma unroll
              for (int j = 0; j < 32; ++j) b[j] = round24(part == 1 ? a[j] : u[j]);
              put_upper(chunk, lane, 32 * q, b);
#pragma unroll
              for (int j = 0; j < 8; ++j) low[8 * q + j] = lower8(b[4 * j], b[4 * j + 1], b[4 * j + 2], b[4 * j + 3]);
            }
          }
          store_chunk<T>(chunk, part == 0 ? &maps.out[0] : &maps.kept[part - 1], nullptr, 0, row, col, p.M, p.N, lane);
        }
        if (p.save) {
          chunk_free(lane);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            *reinterpret_cast<uint4*>(chunk + row64_at(lane, j)) = make_uint4(alow[4 * j], alow[4 * j + 1], alow[4 * j + 2], alow[4 * j + 3]);
            *reinterpret_cast<uint4*>(chunk + kChunkBytes / 2 + row64_at(lane, j)) =
                make_uint4(ulow[4 * j], ulow[4 * j + 1], ulow[4 * j + 2], ulow[4 * j + 3]);
          }
          store_chunk<T>(chunk, &maps.kept[2], nullptr, 0, row, col, p.M, p.N, lane);
          store_chunk<T>(chunk + kChunkBytes / 2, &maps.kept[3], nullptr, 0, row, col, p.M, p.N, lane);
        }
      } else {
        // a piece's a and u go to registers, the next piece's are asked for, and only then the work on them begins: the load's latency
        // and the stores' are both behind it (pieces of 64 columns loaded after the stores before them: 209 us instead of 203, 8192 x 2048 x 5632)
        bool ok = true;
        char* out = chunk + 6144;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          ok = tc::mbar_wait_warp(&sh.loaded[ew], loads & 1, &sh.abort, status, kWaitCode);
          if (!ok) break;
          ++loads;
          float d[32], a[32], u[32];
          tc::tmem_ld32(acc + half * 128 + 32 * c, d);
          get_kept(chunk, chunk + 4096, lane, a);
          get_kept(chunk + 2048, chunk + 5120, lane, u);
          // Every lane's loads of the piece come before the copy that overwrites it: a load from shared memory may wait its turn behind
          // the warps' other accesses for longer than a copy takes to arrive, and neither a warp barrier nor an asm statement without
          // an instruction holds the copy back (an a or u in some tens of calls was the next piece's). Arrivals of all lanes do.
          arrive_read(&sh.read[ew]);
          if (lane == 0 && tc::mbar_wait(&sh.read[ew], (loads - 1) & 1, &sh.abort, status, kWaitCode)) {
            if (c < 3) load_piece(i, c + 1); else load_piece(i + pairs, 0);
          }
          __syncwarp();
          tc::tmem_ld_wait();
          float h[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            float slope;
            const float act = activate<Gelu, true>(a[j], slope);
            h[j] = act * u[j];
            a[j] = d[j] * u[j] * slope;
            u[j] = d[j] * act;
          }
          chunk_free(lane);
          put_row64<T>(out, lane, a);
          put_row64<T>(out + 2048, lane, u);
          put_row64<T>(out + 4096, lane, h);
          tc::fence_async_smem();
          __syncwarp();
          const int col = n * kTile + half * 128 + 32 * c;
          if (lane == 0 && row < p.M && col < p.N) {
            tma_store(&maps.out[0], col, row, tc::smem_u32(out));
            tma_store(&maps.out[1], col, row, tc::smem_u32(out + 2048));
            if (p.save) tma_store(&maps.out[2], col, row, tc::smem_u32(out + 4096));
            tc::bulk_commit();
          }
        }
        if (!ok) break;
      }
      tc::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) arrive_remote(buf ? taken1 : taken0);
      if (buf == 1) phase ^= 1;
      buf ^= 1;
    }
    if (lane == 0) tc::bulk_wait_all();               // nothing reads this block's memory any more
    __syncwarp();
  }
  if constexpr (K == kPlain)
    if (split > 1) join_parts<T>(maps, p, sh, ring, staging, tmem, pair, (int)rank, part, split, status);
  __syncthreads();
  tc::after_a_failure(&sh.abort);
  cluster_sync();                                     // neither block leaves while the other's products or copies need it
  if (wid == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// ---------------------------------------------------------------- few tokens

constexpr int kSkinnyThreads = 256;
constexpr int kMaxSplit = 8;
constexpr int kSkinnyTokens = 128;               // the most tokens of a call that goes this way
constexpr int kSkinnyColumns = 2 * kSkinnyTokens; // of tensor memory: the gate's sums, the up projection's

struct __align__(64) SkinnyMaps {
  CUtensorMap w[2], x;                           // weights (Wg, Wu; or Wd alone) in boxes of 128 rows, tokens in boxes of `width`
};
struct Skinny {
  int steps;                                     // stages of the whole reduction
  int stages, stage_bytes;
  int tokens, width;                             // width: tokens rounded up to 16
  int rows;                                      // weight rows: inner channels, or outputs
  int gelu;
  void* out;
  void* kept;                                    // what a backward pass needs of a and u, or null
  int64_t out_stride, kept_stride;
};

template <typename T, bool Gated>
__global__ void __launch_bounds__(kSkinnyThreads, 2) skinny_kernel(const __grid_constant__ SkinnyMaps maps, const __grid_constant__ Skinny p,
                                                                  uint32_t* status) {
  extern __shared__ __align__(1024) char smem_raw[];
  __shared__ Shared sh;
  char* ring = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int rank = (int)cluster_rank(), CL = (int)gridDim.y;      // the cluster lies along y
  const int row0 = blockIdx.x * kBlockRows;
  const int k0 = (int)((int64_t)p.steps * rank / CL), k1 = (int)((int64_t)p.steps * (rank + 1) / CL);
  constexpr int kWeightBytes = (Gated ? 2 : 1) * kOperandBytes;
  const int token_bytes = p.width * kStep * 2;
  auto fetch_weights = [&](int k, int s) {
    const uint32_t bar = tc::smem_u32(&sh.full[s]), dst = tc::smem_u32(ring + s * p.stage_bytes);
    tc::mbar_expect_tx(&sh.full[s], kWeightBytes + token_bytes);
    tma_load(dst, &maps.w[0], k * kStep, row0, bar);
    if constexpr (Gated) tma_load(dst + kOperandBytes, &maps.w[1], k * kStep, row0, bar);
  };
  auto fetch_tokens = [&](int k, int s) {
    tma_load(tc::smem_u32(ring + s * p.stage_bytes) + kWeightBytes, &maps.x, k * kStep, 0, tc::smem_u32(&sh.full[s]));
  };
  if constexpr (Gated) grid_launch_dependents();      // every block is in place or has been by the time this counts
  const int first = min(p.stages, k1 - k0);           // stages that are asked for before anything else
  if (wid == 0 && lane == 0) {
    for (int i = 0; i < p.stages; ++i) {
      tc::mbar_init(&sh.full[i], 1);
      tc::mbar_init(&sh.empty[i], 1);
    }
    tc::mbar_init(&sh.done[0], 1);
    sh.abort = 0;
    tc::mbar_init_fence();
    tc::fence_async_smem();
    for (int i = 0; i < first; ++i) fetch_weights(k0 + i, i);
    if constexpr (!Gated) grid_wait();                // the tokens are the gated product's results
    for (int i = 0; i < first; ++i) fetch_tokens(k0 + i, i);
  }
  if constexpr (!Gated) grid_wait();
  if (wid == 2) tc::tmem_alloc(&sh.tmem, kSkinnyColumns);
  tc::tc_fence_before_sync();
  __syncthreads();
  tc::tc_fence_after_sync();
  const uint32_t tmem = sh.tmem;

  if (wid == 0) {
    if (lane == 0) {
      int s = first == p.stages ? 0 : first, phase = 0;
      for (int k = k0 + first; k < k1; ++k) {
        if (!tc::mbar_wait(&sh.empty[s], phase, &sh.abort, status, kWaitCode)) break;
        fetch_weights(k, s);
        fetch_tokens(k, s);
        if (++s == p.stages) { s = 0; phase ^= 1; }
      }
    }
    __syncwarp();
  } else if (wid == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_of<T>(false, false, kBlockRows, p.width);
      int s = 0, phase = 0;
      bool ok = true;
      for (int k = k0; k < k1; ++k) {
        if (!tc::mbar_wait(&sh.full[s], phase, &sh.abort, status, kWaitCode)) { ok = false; break; }
        tc::tc_fence_after_sync();
        const uint32_t at = tc::smem_u32(ring + s * p.stage_bytes);
        const uint64_t w = operand_desc<false>(at), x = operand_desc<false>(at + kWeightBytes);
#pragma unroll
        for (int q = 0; q < kStep / 16; ++q) {
          const uint32_t acc = k > k0 || q > 0;
          tc::mma_bf16(tmem, w + q * operand_step<false>(), x + q * operand_step<false>(), idesc, acc);
          if constexpr (Gated)
            tc::mma_bf16(tmem + kSkinnyTokens, w + (kOperandBytes >> 4) + q * operand_step<false>(), x + q * operand_step<false>(), idesc, acc);
        }
        tc::mma_commit(&sh.empty[s]);
        if (++s == p.stages) { s = 0; phase ^= 1; }
      }
      if (ok) tc::mma_commit(&sh.done[0]);
    }
    __syncwarp();
  } else if (wid >= 4) {
    // partial sums to this block's shared memory, [gate | up][token][weight row]; the ring is free: every product has read it
    const int quad = wid & 3;
    float* part = reinterpret_cast<float*>(ring);
    if (tc::mbar_wait_warp(&sh.done[0], 0, &sh.abort, status, kWaitCode)) {
      tc::tc_fence_after_sync();
      for (int n = 0; n < p.width; n += 16) {
#pragma unroll
        for (int g = 0; g < (Gated ? 2 : 1); ++g) {
          float x[16];
          tc::tmem_ld16(tmem + ((uint32_t)(quad * 32) << 16) + g * kSkinnyTokens + n, x);
          tc::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; ++j) part[(g * p.width + n + j) * kBlockRows + quad * 32 + lane] = x[j];
        }
      }
      tc::tc_fence_before_sync();
    }
  }
  __syncthreads();
  tc::after_a_failure(&sh.abort);
  if (CL > 1) cluster_sync();
  // every block finishes its share of the tile's rows for all tokens: the blocks' sums in their order
  {
    const int q0 = 32 * rank / CL, share = 32 * (rank + 1) / CL - q0;         // in groups of four rows
    const uint32_t part = tc::smem_u32(ring);
    uint32_t peer[kMaxSplit];
#pragma unroll
    for (int b = 0; b < kMaxSplit; ++b) peer[b] = in_block(part, b < CL ? b : rank);
    for (int i = tid; i < p.tokens * share; i += kSkinnyThreads) {
      const int n = i / share, r = 4 * (q0 + i - n * share), row = row0 + r;
      if (row >= p.rows) continue;
      float4 x[Gated ? 2 : 1][kMaxSplit], sum[2] = {};
#pragma unroll
      for (int g = 0; g < (Gated ? 2 : 1); ++g)
#pragma unroll
        for (int b = 0; b < kMaxSplit; ++b)
          if (b < CL) {
            float4& f = x[g][b];
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w)
                         : "r"(peer[b] + ((g * p.width + n) * kBlockRows + r) * 4) : "memory");
          }
#pragma unroll
      for (int g = 0; g < (Gated ? 2 : 1); ++g)
#pragma unroll
        for (int b = 0; b < kMaxSplit; ++b)
          if (b < CL) {
            sum[g].x += x[g][b].x; sum[g].y += x[g][b].y; sum[g].z += x[g][b].z; sum[g].w += x[g][b].w;
          }
      const float *v0 = &sum[0].x, *v1 = &sum[1].x;
      T* out = static_cast<T*>(p.out) + (int64_t)n * p.out_stride + row;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (row + k >= p.rows) continue;
        if constexpr (Gated) {
          float none;
          out[k] = from_f32<T>((p.gelu ? activate<true, false>(v0[k], none) : activate<false, false>(v0[k], none)) * v1[k]);
          if (p.kept) {
            const Planes pl = planes(p.kept, p.tokens, p.kept_stride);
            const int64_t e = (int64_t)n * p.kept_stride + row + k;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const uint32_t b = round24(g ? v1[k] : v0[k]);
              pl.upper[g][e] = (uint16_t)(b >> 16);
              pl.lower[g][e] = (uint8_t)(b >> 8);
            }
          }
        } else {
          out[k] = from_f32<T>(v0[k]);
        }
      }
    }
  }
  __syncthreads();
  if (CL > 1) cluster_sync();                         // no block leaves while another reads its sums
  if (wid == 2) tc::tmem_dealloc(tmem, kSkinnyColumns);
}

// ---------------------------------------------------------------- rows to a pitch of 16 bytes

constexpr int kMaxCopies = 6;
struct Copies {
  const uint16_t* src[kMaxCopies];
  uint16_t* dst[kMaxCopies];
  int64_t rows[kMaxCopies], src_stride[kMaxCopies], dst_stride[kMaxCopies];
  int cols[kMaxCopies];
};
// 8 elements a thread, read as the 4-byte words that hold them (a row may start in the middle of one) and shifted into place; what
// lies behind a row's end is zero, and words behind it are not read. Element by element it was bound by its loads: 9.5 us instead of
// 6.5 for the four operands of 1003 x 1001 x 2731.
__global__ void __launch_bounds__(256) align_rows_kernel(const __grid_constant__ Copies c) {
  const int j = blockIdx.y, cols = c.cols[j], per = (cols + 7) / 8;
  const int64_t n = c.rows[j] * per;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / per;
    const int at = (int)(i - r * per) * 8, left = min(cols - at, 8);          // elements of this piece
    const uint16_t* s = c.src[j] + r * c.src_stride[j] + at;
    const int odd = (int)(reinterpret_cast<uintptr_t>(s) >> 1) & 1;
    const uint32_t* word = reinterpret_cast<const uint32_t*>(s - odd);
    const int words = (left + odd + 1) / 2;
    uint32_t w[5], e[4];
#pragma unroll
    for (int q = 0; q < 5; ++q) w[q] = q < words ? __ldg(word + q) : 0u;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      e[q] = odd ? __funnelshift_r(w[q], w[q + 1], 16) : w[q];
      if (2 * q >= left) e[q] = 0u;
      else if (2 * q + 1 >= left) e[q] &= 0xffffu;
    }
    *reinterpret_cast<uint4*>(c.dst[j] + r * c.dst_stride[j] + at) = make_uint4(e[0], e[1], e[2], e[3]);
  }
}

// ---------------------------------------------------------------- host side

// a [rows, cols] matrix of 16-bit elements with rows `stride` elements apart, in boxes of box_rows x 64 (or 32) columns, swizzled over
// the box's row
struct Matrix {
  const void* p;
  int64_t rows, cols, stride;
};
bool make_map(CUtensorMap* map, const Matrix& m, int box_rows, CUtensorMapDataType type, int size, int cols = 64) {
  const EncodeTiled fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows}, strides[1] = {(cuuint64_t)m.stride * size};
  const cuuint32_t box[2] = {(cuuint32_t)cols, (cuuint32_t)box_rows}, unit[2] = {1, 1};
  return fn(map, type, 2, const_cast<void*>(m.p), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
            cols * size == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : cols * size == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool make_map(CUtensorMap* map, const Matrix& m, int box_rows, int dtype, int cols = 64) {
  return make_map(map, m, box_rows, dtype == GDN2_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, cols);
}
// the planes of a kept buffer
bool make_kept_maps(CUtensorMap (&maps)[4], void* kept, const Matrix& h, int cols) {
  const Planes k = planes(kept, h.rows, h.stride);
  for (int g = 0; g < 2; ++g)
    if (!make_map(&maps[g], Matrix{k.upper[g], h.rows, h.cols, h.stride}, 32, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, cols) ||
        !make_map(&maps[2 + g], Matrix{k.lower[g], h.rows, h.cols, h.stride}, 32, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, cols))
      return false;
  return true;
}

bool aligned_rows(const Matrix& m) { return (reinterpret_cast<uintptr_t>(m.p) & 15u) == 0 && m.stride % 8 == 0; }
int steps_of(int64_t k) { return (int)((k + kStep - 1) / kStep); }
int tiles_of(int64_t n, int tile) { return (int)((n + tile - 1) / tile); }

template <typename T, int K, bool A_MN, bool B_MN, bool Gelu = false>
int launch_product(const Maps& maps, const Problem& p, cudaStream_t st) {
  uint32_t* status = device_status_word();
  if (!status) return record_cuda_error(cudaGetLastError());
  auto kernel = product_kernel<T, K, A_MN, B_MN, Gelu>;
  GDN2_CUDA_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem_bytes<K>()));
  const int tiles = p.tiles_m * p.tiles_n, pairs = device_sm_count() / 2, split = K == kPlain ? p.split : 1;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2 * split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * split * (split > 1 || tiles < pairs ? tiles : pairs));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem_bytes<K>();
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  GDN2_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, maps, p, status));
  return GDN2_OK;
}

// Pairs that share a tile's reduction: with few tiles and a long reduction most SMs would idle. A step is 0.27 us of a pair, joining
// the parts 3 us; clusters of 4 and 8 blocks find places for 33 and 15 tiles.
template <typename T, bool A_MN, bool B_MN> int split_of(int tiles, int steps) {
  static ClusterMemo known;
  int best = 1;
  double least = steps * 0.27;
  for (int s = 2; s <= 4; s *= 2) {
    if (steps < 2 * s || tiles > active_clusters(known, reinterpret_cast<const void*>(product_kernel<T, kPlain, A_MN, B_MN, false>), kThreads,
                                                 smem_bytes<kPlain>(), 1, 2 * s))
      continue;
    const double cost = steps * 0.27 / s + 3.0;
    if (cost < least) {
      best = s;
      least = cost;
    }
  }
  return best;
}

#define GDN2_MAP(m, matrix, box)                                     \
  do {                                                               \
    if (!make_map(&(m), matrix, box, dtype)) return GDN2_ERR_UNSUPPORTED; \
  } while (0)

// h (and what is kept of a, u) = the gated product of x and Wg, Wu
template <typename T>
int gated_forward(const Matrix& x, const Matrix& wg, const Matrix& wu, const Matrix& h, void* kept, int gelu, int dtype, cudaStream_t st) {
  Maps maps{};
  Problem p{};
  GDN2_MAP(maps.a[0], x, kBlockRows);
  GDN2_MAP(maps.b[0], wg, kBlockRows);
  GDN2_MAP(maps.b[1], wu, kBlockRows);
  GDN2_MAP(maps.out[0], h, 32);
  if (kept && !make_kept_maps(maps.kept, kept, h, kChunk16)) return GDN2_ERR_UNSUPPORTED;
  p.steps[0] = steps_of(x.cols);
  p.tiles_m = tiles_of(x.rows, kTile);
  p.tiles_n = tiles_of(wg.rows, kBlockRows);
  p.M = (int)x.rows;
  p.N = (int)wg.rows;
  p.save = kept != nullptr;
  return gelu ? launch_product<T, kGated, false, false, true>(maps, p, st) : launch_product<T, kGated, false, false, false>(maps, p, st);
}

// da, du (and h) from dy, Wd and what was kept of a, u
template <typename T>
int gated_backward(const Matrix& dy, const Matrix& wd, void* kept, const Matrix& da, const Matrix& du, const Matrix& h, bool want_h, int gelu,
                   int dtype, cudaStream_t st) {
  Maps maps{};
  Problem p{};
  GDN2_MAP(maps.a[0], dy, kBlockRows);
  GDN2_MAP(maps.b[0], wd, kStep);
  if (!make_kept_maps(maps.kept, kept, h, 32) || !make_map(&maps.out[0], da, 32, dtype, 32) || !make_map(&maps.out[1], du, 32, dtype, 32) ||
      !make_map(&maps.out[2], h, 32, dtype, 32))
    return GDN2_ERR_UNSUPPORTED;
  p.save = want_h;
  p.steps[0] = steps_of(dy.cols);
  p.tiles_m = tiles_of(dy.rows, kTile);
  p.tiles_n = tiles_of(wd.cols, kTile);
  p.M = (int)dy.rows;
  p.N = (int)wd.cols;
  return gelu ? launch_product<T, kGatedBackward, false, true, true>(maps, p, st)
              : launch_product<T, kGatedBackward, false, true, false>(maps, p, st);
}

int set_out(Maps& maps, Problem& p, int part, const Matrix& out, int dtype) {
  p.out_stride = out.stride;
  if (!aligned_rows(out)) p.plain_out[part] = const_cast<void*>(out.p);
  else if (!make_map(&maps.out[part], out, 32, dtype, p.split > 1 ? 32 : 64)) return GDN2_ERR_UNSUPPORTED;
  return GDN2_OK;
}

// out [M, N] = sum over the runs of a_i b_i^T, the operands as they lie: a [M, K] (or [K, M]), b [N, K] (or [K, N])
template <typename T, bool A_MN, bool B_MN>
int product(const Matrix* a, const Matrix* b, int runs, const Matrix& out, int dtype, cudaStream_t st) {
  Maps maps{};
  Problem p{};
  for (int i = 0; i < runs; ++i) {
    GDN2_MAP(maps.a[i], a[i], A_MN ? kStep : kBlockRows);
    GDN2_MAP(maps.b[i], b[i], B_MN ? kStep : kBlockRows);
    p.steps[i] = steps_of(A_MN ? a[i].rows : a[i].cols);
  }
  p.tiles_m = tiles_of(out.rows, kTile);
  p.tiles_n = tiles_of(out.cols, kTile);
  p.split = split_of<T, A_MN, B_MN>(p.tiles_m * p.tiles_n, p.steps[0] + p.steps[1]);
  const int rc = set_out(maps, p, 0, out, dtype);
  if (rc != GDN2_OK) return rc;
  p.M = (int)out.rows;
  p.N = (int)out.cols;
  return launch_product<T, kPlain, A_MN, B_MN>(maps, p, st);
}
// out_i [M, N] = a_i^T b for two a [K, M] and one b [K, N], in one launch
template <typename T>
int two_weight_gradients(const Matrix& a0, const Matrix& a1, const Matrix& b, const Matrix& out0, const Matrix& out1, int dtype, cudaStream_t st) {
  Maps maps{};
  Problem p{};
  GDN2_MAP(maps.a[0], a0, kStep);
  GDN2_MAP(maps.a[1], a1, kStep);
  GDN2_MAP(maps.b[0], b, kStep);
  p.steps[0] = steps_of(b.rows);
  p.split_m = tiles_of(out0.rows, kTile);
  p.tiles_m = 2 * p.split_m;
  p.tiles_n = tiles_of(out0.cols, kTile);
  p.split = split_of<T, true, true>(p.tiles_m * p.tiles_n, p.steps[0]);
  int rc = set_out(maps, p, 0, out0, dtype);
  if (rc == GDN2_OK) rc = set_out(maps, p, 1, out1, dtype);
  if (rc != GDN2_OK) return rc;
  p.M = (int)out0.rows;
  p.N = (int)out0.cols;
  return launch_product<T, kPlain, true, true>(maps, p, st);
}

// For the question how many clusters of two blocks an SM run at one time: of a kernel with tensor memory the runtime says one block an SM,
// whatever it allocates
__global__ void __launch_bounds__(kSkinnyThreads, 2) stand_in_kernel() {}

template <typename T, bool Gated>
int launch_skinny(const Matrix& x, const Matrix& w0, const Matrix* w1, const Matrix& out, void* kept, int64_t kept_stride, int gelu, int dtype,
                  cudaStream_t st) {
  SkinnyMaps maps{};
  Skinny p{};
  p.tokens = (int)x.rows;
  p.width = (p.tokens + 15) / 16 * 16;
  GDN2_MAP(maps.w[0], w0, kBlockRows);
  if (w1) GDN2_MAP(maps.w[1], *w1, kBlockRows);
  GDN2_MAP(maps.x, x, p.width);
  p.steps = steps_of(x.cols);
  p.rows = (int)w0.rows;
  p.gelu = gelu;
  p.out = const_cast<void*>(out.p);
  p.out_stride = out.stride;
  p.kept = kept;
  p.kept_stride = kept_stride;
  p.stage_bytes = (Gated ? 2 : 1) * kOperandBytes + p.width * kStep * 2;
  // Two blocks fit on an SM, so that clusters of any size find places for as many tiles as there are (one block an SM with twice the
  // stages: 15 clusters of 8 run at one time, and the sixteenth tile of a product with 2048 outputs took as long as the other fifteen;
  // one token, 2048 x 5632: 27.5 us against 21.9), as long as each has three stages; with more tokens a block has the SM to itself
  // (64 tokens: 31.8 us with two stages each). As many blocks a tile as there are places for, each with two steps of the
  // reduction at least; over 16 tokens no more than one an SM, because every block brings the tokens, too (replayed from a graph, 24
  // tokens 23.4 us against 23.9; one token 21.9 against 20.9 the other way).
  const int per_sm = 3 * p.stage_bytes <= 110 * 1024 ? 2 : 1;
  const size_t sums = (size_t)(Gated ? 2 : 1) * p.width * kBlockRows * 4;
  p.stages = (per_sm == 2 ? 110 : 220) * 1024 / p.stage_bytes;
  if (p.stages > 8) p.stages = 8;
  size_t smem = (size_t)p.stages * p.stage_bytes;
  smem = (smem > sums ? smem : sums) + 1024;
  auto places = [per_sm](int cl) {
    static ClusterMemo known[2];
    return active_clusters(known[per_sm - 1], reinterpret_cast<const void*>(stand_in_kernel), kSkinnyThreads,
                           (per_sm == 2 ? 112 : 222) * 1024, per_sm, cl);
  };
  const int tiles = tiles_of(w0.rows, kBlockRows);
  int split = kMaxSplit;
  const int blocks = p.width > 16 ? device_sm_count() : 2 * device_sm_count();
  while (split > 1 && (split > p.steps / 2 || tiles > places(split) || tiles * split > blocks)) --split;
  uint32_t* status = device_status_word();
  if (!status) return record_cuda_error(cudaGetLastError());
  auto kernel = skinny_kernel<T, Gated>;
  GDN2_CUDA_TRY(ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem));
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = split;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;      // inside a capture launches stay plain (launch_chained says why)
  const bool chained = !Gated && (cudaStreamIsCapturing(st, &capture) != cudaSuccess || capture == cudaStreamCaptureStatusNone);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tiles, split);
  cfg.blockDim = dim3(kSkinnyThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = chained ? 2 : 1;
  GDN2_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, maps, p, status));
  return GDN2_OK;
}

template <typename T> int forward(const gdn2_ffn_args& f, int dtype, cudaStream_t st) {
  const Matrix x{f.x, f.tokens, f.hidden, f.x_stride}, wg{f.w_gate, f.inner, f.hidden, f.w_gate_stride},
      wu{f.w_up, f.inner, f.hidden, f.w_up_stride}, wd{f.w_down, f.out, f.inner, f.w_down_stride}, h{f.h, f.tokens, f.inner, f.inner_stride},
      y{f.y, f.tokens, f.out, f.y_stride};
  const int gelu = f.activation == GDN2_ACT_GELU_TANH;
  int rc;
  if (f.tokens <= kSkinnyTokens) {
    rc = launch_skinny<T, true>(x, wg, &wu, h, f.kept, f.inner_stride, gelu, dtype, st);
    if (rc != GDN2_OK) return rc;
    return launch_skinny<T, false>(h, wd, nullptr, y, nullptr, 0, 0, dtype, st);
  }
  rc = gated_forward<T>(x, wg, wu, h, f.kept, gelu, dtype, st);
  if (rc != GDN2_OK) return rc;
  return product<T, false, false>(&h, &wd, 1, y, dtype, st);
}

template <typename T> int backward(const gdn2_ffn_args& f, int dtype, cudaStream_t st) {
  const Matrix x{f.x, f.tokens, f.hidden, f.x_stride}, wg{f.w_gate, f.inner, f.hidden, f.w_gate_stride},
      wu{f.w_up, f.inner, f.hidden, f.w_up_stride}, wd{f.w_down, f.out, f.inner, f.w_down_stride}, h{f.h, f.tokens, f.inner, f.inner_stride},
      dy{f.dy, f.tokens, f.out, f.dy_stride},
      da{f.da, f.tokens, f.inner, f.inner_stride}, du{f.du, f.tokens, f.inner, f.inner_stride}, dx{f.dx, f.tokens, f.hidden, f.dx_stride},
      dwg{f.dw_gate, f.inner, f.hidden, f.hidden}, dwu{f.dw_up, f.inner, f.hidden, f.hidden}, dwd{f.dw_down, f.out, f.inner, f.inner};
  int rc = gated_backward<T>(dy, wd, f.kept, da, du, h, f.dw_down != nullptr, f.activation == GDN2_ACT_GELU_TANH, dtype, st);
  if (rc == GDN2_OK && f.dx) {
    const Matrix lhs[2] = {da, du}, rhs[2] = {wg, wu};
    rc = product<T, false, true>(lhs, rhs, 2, dx, dtype, st);
  }
  if (rc == GDN2_OK && f.dw_gate) rc = two_weight_gradients<T>(da, du, x, dwg, dwu, dtype, st);
  if (rc == GDN2_OK && f.dw_down) rc = product<T, true, true>(&dy, &h, 1, dwd, dtype, st);
  return rc;
}

int check(const gdn2_ffn_args& f, int dtype, bool back) {
  if (dtype != GDN2_BF16 && dtype != GDN2_F16) return GDN2_ERR_BAD_DTYPE;
  if (f.activation != GDN2_ACT_SILU && f.activation != GDN2_ACT_GELU_TANH) return GDN2_ERR_UNSUPPORTED;
  const int64_t most = 1LL << 30;
  for (int64_t n : {f.tokens, f.hidden, f.inner, f.out})
    if (n <= 0 || n > most) return GDN2_ERR_BAD_SHAPE;
  // tiles are counted in 32 bits
  if (((f.tokens >> 7) + 1) * ((f.inner >> 6) + 1) > most || ((f.inner >> 7) + 1) * ((f.hidden >> 6) + 1) > most ||
      ((f.tokens >> 7) + 1) * ((f.out >> 6) + 1) > most || ((f.tokens >> 7) + 1) * ((f.hidden >> 6) + 1) > most ||
      ((f.out >> 7) + 1) * ((f.inner >> 6) + 1) > most)
    return GDN2_ERR_BAD_SHAPE;
  if (!f.x || !f.w_gate || !f.w_up || !f.w_down || !f.h) return GDN2_ERR_NULL_POINTER;
  if (back) {
    if (!f.dy || !f.kept || !f.da || !f.du) return GDN2_ERR_NULL_POINTER;
    if ((f.dw_gate == nullptr) != (f.dw_up == nullptr)) return GDN2_ERR_NULL_POINTER;
  } else {
    if (!f.y) return GDN2_ERR_NULL_POINTER;
  }
  if (f.x_stride < f.hidden || f.w_gate_stride < f.hidden || f.w_up_stride < f.hidden || f.w_down_stride < f.inner ||
      f.inner_stride < f.inner || (back ? f.dy_stride < f.out || (f.dx && f.dx_stride < f.hidden) : f.y_stride < f.out))
    return GDN2_ERR_BAD_SHAPE;
  for (int64_t s : {f.x_stride, f.w_gate_stride, f.w_up_stride, f.w_down_stride, f.inner_stride, back ? f.dy_stride : (int64_t)0})
    if (s % 8 || s > (1LL << 34)) return GDN2_ERR_MISALIGNED;
  if (f.inner_stride % 16) return GDN2_ERR_MISALIGNED;        // rows of the byte planes start on 16 bytes, too
  for (const void* q : {f.x, f.w_gate, f.w_up, f.w_down, (const void*)f.h, (const void*)f.kept, back ? f.dy : nullptr,
                        back ? (const void*)f.da : nullptr, back ? (const void*)f.du : nullptr})
    if (reinterpret_cast<uintptr_t>(q) & 15u) return GDN2_ERR_MISALIGNED;
  return GDN2_OK;
}

}  // namespace
}  // namespace gdn2

extern "C" {

size_t gdn2_ffn_kept_bytes(int64_t tokens, int64_t inner_stride) {
  return tokens > 0 && inner_stride > 0 ? (size_t)tokens * (size_t)inner_stride * 6 : 0;
}

int gdn2_ffn_forward(const gdn2_ffn_args* args, int dtype, void* stream) {
  if (!args) return GDN2_ERR_NULL_POINTER;
  int rc = gdn2::check(*args, dtype, false);
  if (rc == GDN2_OK) rc = gdn2::own_context();
  if (rc != GDN2_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == GDN2_BF16 ? gdn2::forward<__nv_bfloat16>(*args, dtype, st) : gdn2::forward<__half>(*args, dtype, st);
}

int gdn2_ffn_backward(const gdn2_ffn_args* args, int dtype, void* stream) {
  if (!args) return GDN2_ERR_NULL_POINTER;
  int rc = gdn2::check(*args, dtype, true);
  if (rc == GDN2_OK) rc = gdn2::own_context();
  if (rc != GDN2_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == GDN2_BF16 ? gdn2::backward<__nv_bfloat16>(*args, dtype, st) : gdn2::backward<__half>(*args, dtype, st);
}

int gdn2_align_rows(const gdn2_row_copy* copies, int64_t n, void* stream) {
  using namespace gdn2;
  if (!copies) return GDN2_ERR_NULL_POINTER;
  if (n < 1 || n > kMaxCopies) return GDN2_ERR_BAD_SHAPE;
  Copies c{};
  int64_t most = 0;
  for (int i = 0; i < n; ++i) {
    const gdn2_row_copy& k = copies[i];
    if (!k.src || !k.dst) return GDN2_ERR_NULL_POINTER;
    if (k.rows < 1 || k.cols < 1 || k.cols > (1LL << 30) || k.rows > (1LL << 30) || k.dst_stride < k.cols || k.src_stride < 0)
      return GDN2_ERR_BAD_SHAPE;
    if ((reinterpret_cast<uintptr_t>(k.dst) & 15u) || k.dst_stride % 8) return GDN2_ERR_MISALIGNED;
    c.src[i] = static_cast<const uint16_t*>(k.src);
    c.dst[i] = static_cast<uint16_t*>(k.dst);
    c.rows[i] = k.rows; c.cols[i] = (int)k.cols; c.src_stride[i] = k.src_stride; c.dst_stride[i] = k.dst_stride;
    const int64_t pieces = k.rows * ((k.cols + 7) / 8);
    most = pieces > most ? pieces : most;
  }
  const int64_t blocks = (most + 255) / 256, cap = 8LL * device_sm_count();
  align_rows_kernel<<<dim3((unsigned)(blocks < cap ? blocks : cap), (unsigned)n), 256, 0, static_cast<cudaStream_t>(stream)>>>(c);
  GDN2_CUDA_TRY(cudaGetLastError());
  return GDN2_OK;
}

}  // extern "C"
