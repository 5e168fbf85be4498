// The int8 product (int8_gemm.cuh) of a few tokens: weights straight from HBM to registers, exact int32 sums.
//
//   out[m, n] = (sum_k x[m, k] * w[n, k]) * x_scales[m] * w_scales[n]        1 <= m <= 8
//
// One or two tokens (rows on 16 bytes): dp4a, four products an instruction.  A weight row belongs to L lanes of a warp, which read 16 L bytes of it at a
// time and have eight such reads each on their way; the lanes' sums meet by shuffles.
//
// Up to eight tokens: warp-level MMAs (m16n8k32), sixteen weight rows by eight tokens.  A lane wants 4 bytes of k of row g, 4 of row g + 8 and 4 of token g.
// Which k they are does not matter as long as weights and tokens agree, so a lane reads sixteen consecutive bytes of each -- four lanes 64 of a row -- and feeds
// them to two MMAs in the order in which they lie.  A row's K is shared by `parts` warps of a block, whose sums meet in shared memory.  Rows may start
// anywhere: ON_16 = false shifts each 16 bytes into place.
//
// Either way the tokens come out of L1, where all rows of an SM's warps find them, and there is no ring to fill, no tensor memory to allocate and no accumulator to
// hand over.  As in int8_gemm.cuh, the first weights are fetched into L2 while the kernel ahead still runs, and read after it has completed.
//
// us, replayed graphs, this / int8_gemm.cuh: 1 x 2048 -> 2048 2.6 / 5.4, 1 x 14336 -> 4096 12.1 / 13.6, 1 x 8192 -> 28672 38.7 / 41;
// 8 x 2048 -> 2048 3.4 / 5.1, 8 x 4096 -> 4096 6.1 / 7.3, 8 x 14336 -> 4096 14.8 / 13.3; rows off 16 bytes (there with their copy): 8 x 4104 -> 28672 42 / 71.
#pragma once
#include "int8_gemm.cuh"

namespace lcq {
namespace int8_gemv {

using int8_gemm::Piece;
constexpr int MAX_M = 8;
constexpr int WARPS = 8;
constexpr int ROWS = 16;                       // weight rows of a warp's MMAs
constexpr int CHUNK = 64;                      // k of a warp's loads for them

struct Params {
  const uint8_t *x, *w;
  long long ldx, ldw;
  const float* x_scales;
  const void* w_scales;
  void* out;
  int M, N, K, w_scale_dtype;
  int parts;                                   // warps that share a row's K: 1, 2, 4 or 8
};

// Streamed once: not kept in L1, where the tokens are.
__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {
  uint4 r;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p) : "memory");
  return r;
}
// 16 bytes of a row, of which the first `valid` count (and the others read as zero).
template <bool ON_16> struct Load;
template <> struct Load<true> {
  uint4 a;
  __device__ __forceinline__ void weights(const uint8_t* p, int valid) { a = valid > 0 ? load_stream(p) : make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void tokens(const uint8_t* p, int valid) { a = valid > 0 ? *reinterpret_cast<const uint4*>(p) : make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ uint4 get(int valid) const {
    if (valid >= 16) return a;
    Piece q;
    q.a = a; q.b = make_uint4(0u, 0u, 0u, 0u); q.off = 0;
    return q.get(valid);
  }
};
template <> struct Load<false> {
  Piece q;
  __device__ __forceinline__ void weights(const uint8_t* p, int valid) { q.load(p, valid); }
  __device__ __forceinline__ void tokens(const uint8_t* p, int valid) { q.load(p, valid); }
  __device__ __forceinline__ uint4 get(int valid) const { return q.get(valid); }
};

template <typename OT, int MT, int L>
__global__ void __launch_bounds__(WARPS * 32) int8_dp4a_kernel(const Params p) {
  constexpr int U = 8, PER_WARP = 32 / L;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % L;
  const int n = (blockIdx.x * WARPS + warp) * PER_WARP + lane / L;
  const bool there = n < p.N;
  const uint8_t* row = p.w + static_cast<long long>(there ? n : p.N - 1) * p.ldw;
  griddep_launch_dependents();
  if (sub % 8 == 0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (sub + u * L) * 16;
      if (there && k < p.K) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + k));
    }
  }
  griddep_wait();
  int acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = 0;
  for (int k0 = sub * 16; k0 < p.K; k0 += U * L * 16) {
    Load<true> w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * L * 16;
      w[u].weights(row + k, k < p.K && there ? p.K - k : 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + u * L * 16;
      if (k >= p.K) break;
      const uint4 wv = w[u].get(there ? p.K - k : 0);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const uint4 xv = *reinterpret_cast<const uint4*>(p.x + m * p.ldx + k);      // (where w reads as zero, x does not matter)
        acc[m] = __dp4a(static_cast<int>(xv.x), static_cast<int>(wv.x), acc[m]);
        acc[m] = __dp4a(static_cast<int>(xv.y), static_cast<int>(wv.y), acc[m]);
        acc[m] = __dp4a(static_cast<int>(xv.z), static_cast<int>(wv.z), acc[m]);
        acc[m] = __dp4a(static_cast<int>(xv.w), static_cast<int>(wv.w), acc[m]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int off = L / 2; off > 0; off >>= 1) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], off);
  }
  if (there && sub < MT) {                     // lane m of the row's lanes writes token m
    int sum = acc[0];
#pragma unroll
    for (int m = 1; m < MT; ++m)
      if (sub == m) sum = acc[m];
    static_cast<OT*>(p.out)[static_cast<long long>(sub) * p.N + n] =
        from_f32<OT>(static_cast<float>(sum) * p.x_scales[sub] * int8_gemm::load_scale(p.w_scales, n, p.w_scale_dtype));
  }
}

// D(16x8, s32) += A(16x32, s8, row) * B(32x8, s8, col)
__device__ __forceinline__ void mma_i8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <typename OT, bool ON_16>
__global__ void __launch_bounds__(WARPS * 32, 3) int8_mma_kernel(const Params p) {
  constexpr int U = ON_16 ? 4 : 2;            // chunks on their way
  __shared__ int sums[WARPS][8][ROWS + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int groups = WARPS / p.parts;          // row groups of a block
  const int row_group = blockIdx.x * groups + warp / p.parts, part = warp % p.parts;
  const int n0 = row_group * ROWS;
  const int chunks = (p.K + CHUNK - 1) / CHUNK;
  const int c0 = static_cast<int>(static_cast<long long>(chunks) * part / p.parts), c1 = static_cast<int>(static_cast<long long>(chunks) * (part + 1) / p.parts);
  const bool there0 = n0 + g < p.N, there1 = n0 + g + 8 < p.N;
  const uint8_t* row0 = p.w + static_cast<long long>(there0 ? n0 + g : p.N - 1) * p.ldw;
  const uint8_t* row1 = p.w + static_cast<long long>(there1 ? n0 + g + 8 : p.N - 1) * p.ldw;
  griddep_launch_dependents();
  {
    const int k = c0 * CHUNK + (t & 1) * 128;
    if (k < p.K && c0 < c1 && (t < 2 ? there0 : there1)) asm volatile("prefetch.global.L2 [%0];" ::"l"((t < 2 ? row0 : row1) + k));
  }
  griddep_wait();
  int acc[4] = {0, 0, 0, 0};
  for (int c = c0; c < c1; c += U) {
    Load<ON_16> w0[U], w1[U], x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (c + u) * CHUNK + t * 16, valid = c + u < c1 ? p.K - k : 0;
      w0[u].weights(row0 + k, there0 ? valid : 0);
      w1[u].weights(row1 + k, there1 ? valid : 0);
      x[u].tokens(p.x + (g < p.M ? g : 0) * p.ldx + k, g < p.M ? valid : 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int valid = c + u < c1 ? p.K - ((c + u) * CHUNK + t * 16) : 0;
      const uint4 a = w0[u].get(there0 ? valid : 0), b = w1[u].get(there1 ? valid : 0), v = x[u].get(g < p.M ? valid : 0);
      mma_i8(acc, a.x, b.x, a.y, b.y, v.x, v.y);
      mma_i8(acc, a.z, b.z, a.w, b.w, v.z, v.w);
    }
  }
  sums[warp][2 * t][g] = acc[0];               // rows g and g + 8, tokens 2 t and 2 t + 1
  sums[warp][2 * t + 1][g] = acc[1];
  sums[warp][2 * t][g + 8] = acc[2];
  sums[warp][2 * t + 1][g + 8] = acc[3];
  __syncthreads();
  for (int i = threadIdx.x; i < groups * ROWS * p.M; i += WARPS * 32) {
    const int r = i % ROWS, m = (i / ROWS) % p.M, group = i / (ROWS * p.M);
    const int n = (blockIdx.x * groups + group) * ROWS + r;
    if (n >= p.N) continue;
    int sum = 0;
    for (int q = 0; q < p.parts; ++q) sum += sums[group * p.parts + q][m][r];
    static_cast<OT*>(p.out)[static_cast<long long>(m) * p.N + n] =
        from_f32<OT>(static_cast<float>(sum) * p.x_scales[m] * int8_gemm::load_scale(p.w_scales, n, p.w_scale_dtype));
  }
}

// ---------------------------------------------------------------------------- host side
template <typename F>
int launch_kernel(F* kern, long long blocks, const Params& p, cudaStream_t st) {
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[1];
  gemm_tc::pdl_launch_config(cfg, attr, static_cast<int>(blocks), WARPS * 32, 0, st);
  LCQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
  return LCQ_OK;
}
template <typename OT>
int launch_t(Params& p, bool on_16, int sm_count, cudaStream_t st) {
  if (p.M <= 2 && on_16) {
    // rows of up to 1024 bytes fill 8 lanes better than 32 (1 x 576 -> 49152: 7.4 us and 15.9; 1 x 2048 -> 8192: 6.5 and 5.0)
    const int lanes = p.K <= 1024 ? 8 : 32;
    const long long per_block = WARPS * (32 / lanes), blocks = (p.N + per_block - 1) / per_block;
    if (lanes == 8) return launch_kernel(p.M == 1 ? int8_dp4a_kernel<OT, 1, 8> : int8_dp4a_kernel<OT, 2, 8>, blocks, p, st);
    return launch_kernel(p.M == 1 ? int8_dp4a_kernel<OT, 1, 32> : int8_dp4a_kernel<OT, 2, 32>, blocks, p, st);
  }
  // eight chunks for a warp where there are that many; more warps to a row where blocks would leave SMs idle (8 x 2048 -> 8192 in 4 parts 6.1 us, in 8 7.0;
  // 8 x 2048 -> 2048 4.2 and 3.4; 8 x 577 -> 49152 in one 14.7, in 4 18.2)
  const int chunks = (p.K + CHUNK - 1) / CHUNK;
  const auto blocks = [&] { return (static_cast<long long>(p.N) + WARPS / p.parts * ROWS - 1) / (WARPS / p.parts * ROWS); };
  p.parts = 1;
  while (p.parts < WARPS && (chunks >= 16 * p.parts || (chunks >= 4 * p.parts && blocks() < sm_count))) p.parts *= 2;
  return launch_kernel(on_16 ? int8_mma_kernel<OT, true> : int8_mma_kernel<OT, false>, blocks(), p, st);
}
// Whether these kernels take the call: one or two tokens, up to eight where little is read (further on the tensor cores' ring streams better, see above) or
// where rows off 16 bytes would have to be copied.  Not one or two tokens of many rows of 1025 .. 4095 bytes: a warp's loads reach over 4096 bytes, and what they have on
// their way of such a row is less.  us in graphs, this / ring: 1 x 1536 -> 28672 11.1 / 9.2, -> 151936 51 / 38; 1 x 2048 -> 16384 8.7 / 8.6, -> 49152 19.6 / 17.9;
// 1 x 2560 -> 151936 69 / 60; but 1 x 2048 -> 8192 5.0 / 6.8, 1 x 1024 -> 65536 12.2 / 12.8, 1 x 4096 -> 49152 30.6 / 33.3, 1 x 8192 -> 28672 33 / 41.
inline bool takes(int M, int N, int K, bool on_16) {
  const long long bytes = static_cast<long long>(N) * K;
  if (M <= 2) return !on_16 || K <= 1024 || K >= 4096 || bytes < (32ll << 20);
  return M <= MAX_M && (!on_16 || (K <= 4096 && bytes <= (20ll << 20)));
}
inline int launch(const int8_gemm::Operands& o, int M, int N, int K, int sm_count, cudaStream_t st) {
  Params p = {static_cast<const uint8_t*>(o.x), static_cast<const uint8_t*>(o.w), o.ldx, o.ldw, o.x_scales, o.w_scales, o.out, M, N, K, o.w_scale_dtype, 1};
  const bool on_16 = int8_gemm::mappable(o.x, o.ldx) && int8_gemm::mappable(o.w, o.ldw);
  switch (o.out_dtype) {
    case LCQ_F32: return launch_t<float>(p, on_16, sm_count, st);
    case LCQ_F16: return launch_t<__half>(p, on_16, sm_count, st);
    case LCQ_BF16: return launch_t<__nv_bfloat16>(p, on_16, sm_count, st);
    default: break;
  }
  set_error("int8 matmul: bad out_dtype %d", o.out_dtype);
  return LCQ_ERR_BAD_ARG;
}

}  // namespace int8_gemv
}  // namespace lcq
