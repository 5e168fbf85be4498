// The int8 product (int8_gemm.cuh) of a few tokens on CUDA cores: four products an instruction (dp4a), weights straight from HBM to registers.
//
//   out[m, n] = (sum_k x[m, k] * w[n, k]) * x_scales[m] * w_scales[n]        1 <= m <= 8, exact int32 sums
//
// A weight row belongs to L lanes of a warp, which read 16 L bytes of it at a time and have U such reads each on their way; the tokens come
// out of L1, where all rows of an SM's warps find them.  The lanes' sums meet by shuffles.  There is no ring to fill, no tensor memory to
// allocate and no accumulator to hand over.  Rows may start anywhere: ON_16 = false shifts each 16 bytes into place.
// As in int8_gemm.cuh, the first weights are fetched into L2 while the kernel ahead still runs, and read after it has completed.
#pragma once
#include "int8_gemm.cuh"

namespace lcq {
namespace int8_gemv {

using int8_gemm::Piece;
constexpr int MAX_M = 8;
constexpr int WARPS = 8;

struct Params {
  const uint8_t *x, *w;
  long long ldx, ldw;
  const float* x_scales;
  const void* w_scales;
  void* out;
  int M, N, K, w_scale_dtype;
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
  __device__ __forceinline__ void tokens(const uint8_t* p, int) { a = *reinterpret_cast<const uint4*>(p); }
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

template <typename OT, int MT, int L, bool ON_16>
__global__ void __launch_bounds__(WARPS * 32) int8_gemv_kernel(const Params p) {
  constexpr int U = ON_16 ? (MT <= 2 ? 8 : 4) : (MT <= 2 ? 4 : 2), ROWS = 32 / L;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % L;
  const int n = (blockIdx.x * WARPS + warp) * ROWS + lane / L;
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
    Load<ON_16> w[U];
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
        if (MT > 2 && m >= p.M) break;
        Load<ON_16> x;
        x.tokens(p.x + m * p.ldx + k, p.K - k);
        const uint4 xv = ON_16 ? x.get(16) : x.get(p.K - k);      // (where w reads as zero, x does not matter)
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
  if (there && sub < MT && sub < p.M) {        // lane m of the row's lanes writes token m
    int sum = acc[0];
#pragma unroll
    for (int m = 1; m < MT; ++m)
      if (sub == m) sum = acc[m];
    static_cast<OT*>(p.out)[static_cast<long long>(sub) * p.N + n] =
        from_f32<OT>(static_cast<float>(sum) * p.x_scales[sub] * int8_gemm::load_scale(p.w_scales, n, p.w_scale_dtype));
  }
}

template <typename OT, int MT, int L, bool ON_16>
int launch_t(const Params& p, cudaStream_t st) {
  const long long per_block = WARPS * (32 / L), blocks = (p.N + per_block - 1) / per_block;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[1];
  gemm_tc::pdl_launch_config(cfg, attr, static_cast<int>(blocks), WARPS * 32, 0, st);
  LCQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, int8_gemv_kernel<OT, MT, L, ON_16>, p));
  return LCQ_OK;
}
// Rows of up to 1024 bytes fill 8 lanes better than 32 (1 x 576 -> 49152: 7.4 us and 15.9; 1 x 2048 -> 8192: 6.5 and 5.0).
template <typename OT, bool ON_16>
int launch_m(const Params& p, cudaStream_t st) {
  if (p.M <= 2 && p.K <= 1024) return p.M == 1 ? launch_t<OT, 1, 8, ON_16>(p, st) : launch_t<OT, 2, 8, ON_16>(p, st);
  if (p.M <= 2) return p.M == 1 ? launch_t<OT, 1, 32, ON_16>(p, st) : launch_t<OT, 2, 32, ON_16>(p, st);
  return p.M <= 4 ? launch_t<OT, 4, 32, ON_16>(p, st) : launch_t<OT, 8, 32, ON_16>(p, st);
}
// Whether this kernel takes the call.  Up to two tokens it streams weights as fast as TMA or faster and starts sooner (us here / there: 1 x 8192 -> 28672
// 34.5 / 42.5, 1 x 14336 -> 4096 12.2 / 13.6, 2 x 8192 -> 28672 37.2 / 43.4, 1 x 2048 -> 49152 20.5 / 19.8); with more, reading the tokens bounds it (4 x 8192 -> 28672
// 55.8 / 43.2), and only small products come out ahead -- larger ones where rows off 16 bytes would have to be copied.
inline bool takes(int M, int N, int K, bool on_16) {
  if (M <= 2) return true;
  return M <= MAX_M && static_cast<double>(M) * N * K <= (on_16 ? 8e6 : 20e6);
}
inline int launch(const int8_gemm::Operands& o, int M, int N, int K, cudaStream_t st) {
  Params p = {static_cast<const uint8_t*>(o.x), static_cast<const uint8_t*>(o.w), o.ldx, o.ldw, o.x_scales, o.w_scales, o.out, M, N, K, o.w_scale_dtype};
  const bool on_16 = int8_gemm::mappable(o.x, o.ldx) && int8_gemm::mappable(o.w, o.ldw);
  switch (o.out_dtype) {
    case LCQ_F32: return on_16 ? launch_m<float, true>(p, st) : launch_m<float, false>(p, st);
    case LCQ_F16: return on_16 ? launch_m<__half, true>(p, st) : launch_m<__half, false>(p, st);
    case LCQ_BF16: return on_16 ? launch_m<__nv_bfloat16, true>(p, st) : launch_m<__nv_bfloat16, false>(p, st);
    default: break;
  }
  set_error("int8 matmul: bad out_dtype %d", o.out_dtype);
  return LCQ_ERR_BAD_ARG;
}

}  // namespace int8_gemv
}  // namespace lcq
