// What stands between the int8 products of a decoder layer, a row (token) at a time:
//
//   ROWS      v = x, or x * rsqrt(mean(x^2) + eps) * weight
//   SILU_MUL  v = gate * sigmoid(gate) * up
//   RESIDUAL  y = delta, or delta * rsqrt(mean(delta^2) + eps) * post_weight;  y *= gate
//             hidden_out = hidden + scale * y, rounded to the storage type;  v = hidden_out * rsqrt(mean(hidden_out^2) + eps) * weight
//
// and v goes out in the storage type (RESIDUAL), or as int8 with a float32 scale for the row:
//   s = max |v| / 127 (at least 2^-126; 1 for a row of zeros), q = rint(v / s).
// A row that holds an infinity or NaN gets the scale NaN and q = 0, so that every product with it is NaN, and no other row's.
// All arithmetic is float32.  Without a norm s and q are bit for bit those of the weight quantiser with the row as its group.
// With one, the factor rsqrt(..) is common to v and s: q is taken from the products with the weight alone, and one reduction finds
// their maximum together with the sum of squares.
//
// HBM-bound; each value is read once and kept in registers from the first load to the last use.  A row belongs to a block of
// as many threads as it has groups of E octets, or to a warp where it is short; all of a thread's loads are issued before the
// first reduction.  Rows longer than a block holds are walked in chunks and read again (from L2) for each pass over them.
#pragma once
#include "common.cuh"
#include "glue.cuh"
#include "quantize.cuh"

namespace lcq {
namespace rows {

enum Op { ROWS, SILU_MUL, RESIDUAL };

struct Args {
  const void *a, *b;           // ROWS: x; SILU_MUL: gate, up; RESIDUAL: hidden, delta
  long long lda, ldb;          // elements between rows
  const void* weight;          // RESIDUAL, and ROWS with a norm
  const void* post_weight;     // RESIDUAL: may be null
  const void* gate;            // RESIDUAL: may be null; [gate_rows, n]
  long long rows_per_gate;
  void* hidden_out;
  void* out;                   // q (int8), or v in the storage type; null: none (RESIDUAL without `weight`)
  long long ldo;               // elements between rows of out
  float* scales;
  long long n_rows;
  int n;
  float eps, scale;
};

// Eight values of a row as they are stored: consecutive ones (VEC), or every `step`-th.
template <typename T, bool VEC> struct Octet;
template <typename T> struct Octet<T, true> {
  uint4 r[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p, int, int) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const { glue::load_vec8<T>(reinterpret_cast<const T*>(r), v); }
  __device__ __forceinline__ void set(const float (&v)[8]) { glue::store_vec8<T>(reinterpret_cast<T*>(r), v); }
  __device__ __forceinline__ void store(T* p, int, int) const {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4*>(p)[i] = r[i];
  }
};
template <typename T> struct Octet<T, false> {
  T r[8];
  __device__ __forceinline__ void load(const T* p, int step, int left) {      // left: values from p on that exist
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = j * step < left ? p[j * step] : from_f32<T>(0.0f);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = from_f32<T>(0.0f);
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32<T>(r[j]);
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = from_f32<T>(v[j]);
  }
  __device__ __forceinline__ void store(T* p, int step, int left) const {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * step < left) p[j * step] = r[j];
  }
};

// Sum of s and maximum of m (bits of a magnitude: NaN above infinity above the numbers) over the threads of a row.
template <bool WARP_ROW>
__device__ __forceinline__ void reduce_row(float& s, uint32_t& m, float2* red) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, off);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, off));
  }
  if (WARP_ROW) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  if (lane == 0) red[warp] = make_float2(s, __uint_as_float(m));
  __syncthreads();
  const float2 t = lane < nw ? red[lane] : make_float2(0.0f, 0.0f);
  s = t.x;
  m = __float_as_uint(t.y);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, off);
    m = max(m, __shfl_xor_sync(0xffffffffu, m, off));
  }
}

__device__ __forceinline__ float silu_mul(float g, float u) { return (g * (1.0f / (1.0f + expf(-g)))) * u; }

// q[j] = rint(v[j] / s): the product with 1 / s gives the same integer unless it comes near a half-integer (quantize.cuh).
template <bool VEC>
__device__ __forceinline__ void store_q(int8_t* p, int step, int left, const float (&v)[8], float s, float inv, bool finite) {
  uint32_t bits[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float t = v[j] * inv;
    float r = t + quant::ROUND_MAGIC;
    if (fabsf(t - (r - quant::ROUND_MAGIC)) > quant::round_limit<8>()) r = rintf(__fdiv_rn(v[j], s)) + quant::ROUND_MAGIC;
    bits[j] = finite ? __float_as_uint(r) : 0u;
  }
  if (VEC) {
    const uint2 o = quant::pack_octet<8>(bits);
    *reinterpret_cast<uint2*>(p) = o;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * step < left) p[j * step] = static_cast<int8_t>(bits[j]);
  }
}

template <typename T, int OP, bool QUANT, bool VEC, int E, bool WARP_ROW, bool WHOLE>
__global__ void __launch_bounds__(WARP_ROW ? 128 : WHOLE ? 1024 : 512) rows_kernel(const Args p) {
  __shared__ float2 red[2][32];
  griddep_launch_dependents();
  griddep_wait();
  const long long row = WARP_ROW ? static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP_ROW && row >= p.n_rows) return;
  const int t = WARP_ROW ? threadIdx.x & 31 : threadIdx.x, T_ROW = WARP_ROW ? 32 : blockDim.x;
  const int step = VEC ? 1 : T_ROW, per_octet = 8 * T_ROW, per_chunk = E * per_octet;
  const int i0 = VEC ? t * 8 : t;                    // this thread's first value in an octet group
  const T* a = static_cast<const T*>(p.a) + row * p.lda;
  const T* b = static_cast<const T*>(p.b) + row * p.ldb;
  const T* gate = static_cast<const T*>(p.gate);
  if (OP == RESIDUAL && gate) gate += row / p.rows_per_gate * p.n;
  const T* weight = static_cast<const T*>(p.weight);
  const T* post = static_cast<const T*>(p.post_weight);
  T* hidden = static_cast<T*>(p.hidden_out) + row * p.n;
  const bool normed = OP == RESIDUAL || (OP == ROWS && weight);

  Octet<T, VEC> x[E], y[E];                          // RESIDUAL: hidden, delta
  const auto fetch = [&](Octet<T, VEC>(&o)[E], const T* src, int c0) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = c0 + e * per_octet + i0;
      if (i < p.n) o[e].load(src + i, step, p.n - i);
      else o[e].zero();
    }
  };
  if (WHOLE) {
    fetch(x, a, 0);
    if (OP != ROWS) fetch(y, b, 0);
  }

  float rd = 1.0f;                                   // RESIDUAL: 1 / rms of delta
  if (OP == RESIDUAL && post) {
    float ss = 0.0f;
    uint32_t none = 0u;
    for (int c0 = 0; c0 < (WHOLE ? 1 : p.n); c0 += per_chunk) {
      if (!WHOLE) fetch(y, b, c0);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float v[8];
        y[e].get(v);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
      }
    }
    reduce_row<WARP_ROW>(ss, none, red[0]);
    rd = rsqrtf(ss / static_cast<float>(p.n) + p.eps);
  }

  float ss = 0.0f;
  uint32_t amax = 0u;
  const auto magnitude = [&](float v) { amax = max(amax, __float_as_uint(fabsf(v))); };
  for (int c0 = 0; c0 < (WHOLE ? 1 : p.n); c0 += per_chunk) {
    if (!WHOLE) {
      fetch(x, a, c0);
      if (OP != ROWS) fetch(y, b, c0);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = c0 + e * per_octet + i0;
      if (i >= p.n) continue;
      float v[8], u[8];
      x[e].get(v);
      if (OP == SILU_MUL) {
        y[e].get(u);
#pragma unroll
        for (int j = 0; j < 8; ++j) magnitude(silu_mul(v[j], u[j]));
        continue;
      }
      if (OP == RESIDUAL) {
        y[e].get(u);
        Octet<T, VEC> o;
        float f[8];
        if (post) {
          o.load(post + i, step, p.n - i);
          o.get(f);
#pragma unroll
          for (int j = 0; j < 8; ++j) u[j] = u[j] * rd * f[j];
        }
        if (gate) {
          o.load(gate + i, step, p.n - i);
          o.get(f);
#pragma unroll
          for (int j = 0; j < 8; ++j) u[j] *= f[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = fmaf(p.scale, u[j], v[j]);
        x[e].set(v);                                 // the value that is stored, which the norm reads
        x[e].store(hidden + i, step, p.n - i);
        x[e].get(v);
      }
      if (normed) {
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
        if (QUANT) {
          Octet<T, VEC> o;
          o.load(weight + i, step, p.n - i);
          o.get(u);
#pragma unroll
          for (int j = 0; j < 8; ++j) magnitude(v[j] * u[j]);
        }
      } else if (QUANT) {
#pragma unroll
        for (int j = 0; j < 8; ++j) magnitude(v[j]);
      }
    }
  }
  if (!QUANT && !weight) return;                     // RESIDUAL without a norm after it
  reduce_row<WARP_ROW>(ss, amax, red[1]);
  const float rr = normed ? rsqrtf(ss / static_cast<float>(p.n) + p.eps) : 1.0f;
  const bool finite = amax < 0x7F800000u;
  // the row's scale, without the factor rr
  const float s = amax == 0u ? 1.0f : fmaxf(__fdiv_rn(__uint_as_float(amax), 127.0f), 1.17549435e-38f);
  const float inv = __fdiv_rn(1.0f, s);
  if (QUANT && t == 0) p.scales[row] = !finite ? __uint_as_float(0x7FC00000u) : amax == 0u ? 1.0f : normed ? s * rr : s;

  for (int c0 = 0; c0 < (WHOLE ? 1 : p.n); c0 += per_chunk) {
    if (!WHOLE) {
      fetch(x, OP == RESIDUAL ? hidden : a, c0);     // (each thread reads what it has written itself)
      if (OP == SILU_MUL) fetch(y, b, c0);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = c0 + e * per_octet + i0;
      if (i >= p.n) continue;
      float v[8], u[8];
      x[e].get(v);
      if (OP == SILU_MUL) {
        y[e].get(u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = silu_mul(v[j], u[j]);
      } else if (normed) {
        Octet<T, VEC> o;
        o.load(weight + i, step, p.n - i);
        o.get(u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = QUANT ? v[j] * u[j] : v[j] * rr * u[j];
      }
      if (QUANT) {
        store_q<VEC>(static_cast<int8_t*>(p.out) + row * p.ldo + i, step, p.n - i, v, s, inv, finite);
      } else {
        Octet<T, VEC> o;
        o.set(v);
        o.store(static_cast<T*>(p.out) + row * p.ldo + i, step, p.n - i);
      }
    }
  }
}

// ---------------------------------------------------------------------------- host side
template <typename T, int OP, bool QUANT, bool VEC, int E, bool WARP_ROW, bool WHOLE>
int launch_form(const Args& p, int threads, cudaStream_t st) {
  const long long blocks = WARP_ROW ? (p.n_rows + 3) / 4 : p.n_rows;
  if (blocks > 2147483647LL) { set_error("too many rows"); return LCQ_ERR_UNSUPPORTED; }
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[1];
  glue::pdl_config(cfg, attr, dim3(static_cast<unsigned>(blocks)), dim3(threads), st);
  LCQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, rows_kernel<T, OP, QUANT, VEC, E, WARP_ROW, WHOLE>, p));
  return LCQ_OK;
}
template <typename T, int OP, bool QUANT, bool VEC>
int launch_vec(const Args& p, cudaStream_t st) {
  const auto threads = [&](int e) { return ((p.n + 8 * e - 1) / (8 * e) + 31) / 32 * 32; };
  if (p.n <= 512 && p.n_rows >= 4) return launch_form<T, OP, QUANT, VEC, 2, true, true>(p, 128, st);
  if (p.n <= 8192) return launch_form<T, OP, QUANT, VEC, 1, false, true>(p, threads(1), st);
  if (p.n <= 16384) return launch_form<T, OP, QUANT, VEC, 2, false, true>(p, threads(2), st);
  return launch_form<T, OP, QUANT, VEC, 2, false, false>(p, 512, st);
}
// Octets of consecutive values where every row of every operand starts on 16 bytes (of q: on 8).
template <typename T, int OP, bool QUANT>
int launch(const Args& p, cudaStream_t st) {
  const auto rows_on_16 = [&](const void* q, long long ld) { return aligned(q, 16) && (ld * sizeof(T)) % 16 == 0; };
  const bool vec = p.n % 8 == 0 && rows_on_16(p.a, p.lda) && rows_on_16(p.b, p.ldb) && aligned(p.weight, 16) && aligned(p.post_weight, 16) &&
                   aligned(p.gate, 16) && aligned(p.hidden_out, 16) &&
                   (QUANT ? aligned(p.out, 8) && p.ldo % 8 == 0 : rows_on_16(p.out, p.ldo));
  return vec ? launch_vec<T, OP, QUANT, true>(p, st) : launch_vec<T, OP, QUANT, false>(p, st);
}

}  // namespace rows
}  // namespace lcq
