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
// delta may be float32 where hidden is 16 bits wide: a product's result that is normalised and added here need not be rounded between.
// All arithmetic is float32.  Without a norm s and q are bit for bit those of the weight quantiser with the row as its group.
// With one, the factor rsqrt(..) is common to v and s: q is taken from the products with the weight alone, and one reduction finds
// their maximum together with the sum of squares.
//
// HBM-bound; each value is read once and kept in registers from the first load to the last use.  A row belongs to a block of as many threads as
// it has groups of E octets (8 consecutive values), or to a warp where it is short; all of a thread's loads are issued before the first reduction.
// Rows longer than a block holds are walked in chunks and read again (from L2) for each pass over them.
// ALIGNED = false: rows start anywhere and have any length.  Octets then begin where the row that is written lies on 16 bytes, so that only the first and the last
// one are stored value by value; what is read lies in two (float32: three) aligned pieces, whose values are shifted into place.
#pragma once
#include "common.cuh"
#include "glue.cuh"
#include "quantize.cuh"

namespace lcq {
namespace rows {

enum Op { ROWS, NORM_ROWS, SILU_MUL, RESIDUAL };

struct Args {
  const void *a, *b;           // ROWS, NORM_ROWS: x; SILU_MUL: gate, up; RESIDUAL: hidden, delta
  long long lda, ldb;          // elements between rows
  const void* weight;          // NORM_ROWS; RESIDUAL: may be null
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

// Eight values as they are stored.
template <typename T> struct Octet {
  static constexpr int W = sizeof(T) / 2;            // 16-byte pieces
  uint4 r[W];
  __device__ __forceinline__ void get(float (&v)[8]) const { glue::load_vec8<T>(reinterpret_cast<const T*>(r), v); }
  __device__ __forceinline__ void set(const float (&v)[8]) { glue::store_vec8<T>(reinterpret_cast<T*>(r), v); }
  // Values i .. i + 7 of a row of n, those there are.
  template <bool ALIGNED> __device__ __forceinline__ void store(T* row, int i, int n) const {
    T* p = row + i;
    if (ALIGNED || (i >= 0 && i + 8 <= n && (reinterpret_cast<uintptr_t>(p) & 15) == 0)) {
#pragma unroll
      for (int j = 0; j < W; ++j) reinterpret_cast<uint4*>(p)[j] = r[j];
    } else {
      float v[8];
      get(v);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i + j >= 0 && i + j < n) p[j] = from_f32<T>(v[j]);
    }
  }
};
// The same on their way from memory: the aligned pieces they lie in.
template <typename T, bool ALIGNED> struct Raw {
  static constexpr int W = Octet<T>::W;
  uint4 r[W];
  __device__ __forceinline__ void load(const T* row, int i, int) {
#pragma unroll
    for (int j = 0; j < W; ++j) r[j] = reinterpret_cast<const uint4*>(row + i)[j];
  }
  __device__ __forceinline__ Octet<T> octet(const T*, int, int) const {
    Octet<T> o;
#pragma unroll
    for (int j = 0; j < W; ++j) o.r[j] = r[j];
    return o;
  }
};
template <typename T> struct Raw<T, false> {
  static constexpr int W = Octet<T>::W, S = sizeof(T);
  uint4 r[W + 1];
  // Only pieces that hold one of the values 0 .. n - 1 are read.
  __device__ __forceinline__ void load(const T* row, int i, int n) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(row) + static_cast<long long>(i) * S;
    const int off = static_cast<int>(p & 15);
    const int first = off + (i < 0 ? -i : 0) * S, end = off + (n - i < 8 ? n - i : 8) * S;
    const uint4* q = reinterpret_cast<const uint4*>(p - off);
#pragma unroll
    for (int j = 0; j <= W; ++j) r[j] = 16 * j < end && 16 * (j + 1) > first ? q[j] : make_uint4(0u, 0u, 0u, 0u);
  }
  // The values in place; those that do not exist are zero.
  __device__ __forceinline__ Octet<T> octet(const T* row, int i, int n) const {
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row) + static_cast<long long>(i) * S) & 15);
    uint32_t w[4 * W + 4];
#pragma unroll
    for (int j = 0; j <= W; ++j) { w[4 * j] = r[j].x; w[4 * j + 1] = r[j].y; w[4 * j + 2] = r[j].z; w[4 * j + 3] = r[j].w; }
    if (S == 4 || off) {                             // (the same for a whole row; in float32 the branch costs registers that are short)
      if (off & 8) {
#pragma unroll
        for (int j = 0; j < 4 * W + 2; ++j) w[j] = w[j + 2];
      }
      if (off & 4) {
#pragma unroll
        for (int j = 0; j < 4 * W + 1; ++j) w[j] = w[j + 1];
      }
      if (S == 2) {
#pragma unroll
        for (int j = 0; j < 4 * W; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], (off & 2) * 8);
      }
    }
    if (i < 0 || i + 8 > n) {
#pragma unroll
      for (int j = 0; j < 4 * W; ++j) {
        const int k = i + j * (4 / S);               // the word's first value
        uint32_t keep = S == 4 ? (k >= 0 && k < n ? 0xFFFFFFFFu : 0u) : (k >= 0 && k < n ? 0xFFFFu : 0u) | (k + 1 >= 0 && k + 1 < n ? 0xFFFF0000u : 0u);
        w[j] &= keep;
      }
    }
    Octet<T> o;
#pragma unroll
    for (int j = 0; j < W; ++j) o.r[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    return o;
  }
};

// Eight values at a time.  PAIRS: two an instruction, since instructions bound these rows as much as memory does; one by one where registers are short.
template <bool PAIRS> __device__ __forceinline__ void mul8(float (&a)[8], const float (&b)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 r = PAIRS ? unpack_pair(mul_pair(pack_pair(a[j], a[j + 1]), pack_pair(b[j], b[j + 1]))) : make_float2(a[j] * b[j], a[j + 1] * b[j + 1]);
    a[j] = r.x;
    a[j + 1] = r.y;
  }
}
template <bool PAIRS> __device__ __forceinline__ void scale8(float (&a)[8], float s) {
  const float t[8] = {s, s, s, s, s, s, s, s};
  mul8<PAIRS>(a, t);
}
template <bool PAIRS> __device__ __forceinline__ void add_scaled8(float (&v)[8], float s, const float (&u)[8]) {      // v += s * u
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const float2 r = PAIRS ? unpack_pair(fma_pair(pack_pair(s, s), pack_pair(u[j], u[j + 1]), pack_pair(v[j], v[j + 1])))
                           : make_float2(fmaf(s, u[j], v[j]), fmaf(s, u[j + 1], v[j + 1]));
    v[j] = r.x;
    v[j + 1] = r.y;
  }
}
// Two sums, the same ones either way.  A row in chunks adds each chunk's to a double, so that the error does not grow with the row: at most 32 squares meet in
// float32 before the tree of shuffles, whatever its length (2^24 values of 0.7 in one float32 sum a thread: the norm 1.1e-4 off).
struct Squares {
  double chunks = 0.0;
  uint64_t two = 0;
  float one = 0.0f, other = 0.0f;
  template <bool PAIRS> __device__ __forceinline__ void add(const float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      if (PAIRS) {
        const uint64_t p = pack_pair(v[j], v[j + 1]);
        two = fma_pair(p, p, two);
      } else {
        one = fmaf(v[j], v[j], one);
        other = fmaf(v[j + 1], v[j + 1], other);
      }
    }
  }
  template <bool PAIRS> __device__ __forceinline__ float sum() const {
    const float2 r = unpack_pair(two);
    return PAIRS ? r.x + r.y : one + other;
  }
  template <bool PAIRS> __device__ __forceinline__ void end_chunk() {
    chunks += static_cast<double>(sum<PAIRS>());
    two = 0;
    one = other = 0.0f;
  }
  template <bool PAIRS, bool WHOLE> __device__ __forceinline__ float total() const { return WHOLE ? sum<PAIRS>() : static_cast<float>(chunks); }
};

// The larger magnitude, or NaN where there is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sum of s and maximum of m over the threads of a row.
template <bool WARP_ROW>
__device__ __forceinline__ void reduce_row(float& s, float& m, float2* red) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, off);
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, off));
  }
  if (WARP_ROW) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  if (lane == 0) red[warp] = make_float2(s, m);
  __syncthreads();
  const float2 t = lane < nw ? red[lane] : make_float2(0.0f, 0.0f);
  s = t.x;
  m = t.y;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, off);
    m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, off));
  }
}
template <bool WARP_ROW>
__device__ __forceinline__ void reduce_row(float& s, float2* red) {
  float none = 0.0f;
  reduce_row<WARP_ROW>(s, none, red);
}

// (the reciprocal is good to one unit in the last place: within the bound of the product's other roundings)
__device__ __forceinline__ float silu_mul(float g, float u) { return (g * quant::approx_rcp(1.0f + expf(-g))) * u; }

// q[j] = rint(v[j] / s), inv = 1 / s.  Adding 1.5 * 2^23 to the exact product rounds it to an integer.  EXACT: bit for bit the quotient's, for which octets
// with a product near a half-integer are divided (quantize.cuh).  ROUNDED: the product is rounded to float32 first, as a quotient would be.  Norms of 16-bit values
// want it: their products with the weight are a few bits long, so that quotients that are half-integers are common, and unrounded products fall to the side that
// the rounding of inv chose, for a whole row (of amax / 2 over all 8-bit amax 48 % wrongly; rounded 12 %, divided 15 %).  It costs 1 to 3 % (8192 x 8192
// NORM_ROWS 37.2 and 38.4; dividing near half-integers 51).  finite = false: zeros.
template <bool ALIGNED, bool EXACT, bool ROUNDED>
__device__ __forceinline__ void store_q(int8_t* row, int i, int n, const float (&v)[8], float s, float inv, bool finite) {
  uint32_t bits[8];
  float off = 0.0f;                                  // how far the products are from their integers, at most
  const uint64_t inv2 = pack_pair(inv, inv), magic2 = pack_pair(quant::ROUND_MAGIC, quant::ROUND_MAGIC), minus2 = pack_pair(-1.0f, -1.0f), one2 = pack_pair(1.0f, 1.0f);
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const uint64_t v2 = pack_pair(v[j], v[j + 1]), r2 = ROUNDED ? fma_pair(mul_pair(v2, inv2), one2, magic2) : fma_pair(v2, inv2, magic2);
    const float2 r = unpack_pair(r2);
    if (EXACT) {
      const float2 d = unpack_pair(fma_pair(v2, inv2, fma_pair(r2, minus2, magic2)));
      off = fmaxf(off, fmaxf(fabsf(d.x), fabsf(d.y)));
    }
    bits[j] = __float_as_uint(r.x);
    bits[j + 1] = __float_as_uint(r.y);
  }
  if (EXACT && off > quant::round_limit<8>()) {
#pragma unroll
    for (int j = 0; j < 8; ++j) bits[j] = __float_as_uint(rintf(__fdiv_rn(v[j], s)) + quant::ROUND_MAGIC);
  }
  uint2 o = quant::pack_octet<8>(bits);
  if (!finite) o = make_uint2(0u, 0u);
  int8_t* p = row + i;
  if (ALIGNED || (i >= 0 && i + 8 <= n && (reinterpret_cast<uintptr_t>(p) & 7) == 0)) {
    *reinterpret_cast<uint2*>(p) = o;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j >= 0 && i + j < n) p[j] = static_cast<int8_t>((j < 4 ? o.x : o.y) >> (8 * (j & 3)));
  }
}

// E octets a thread; WARP_ROW: four rows a block, a warp each; WHOLE: a row fits into the registers of its threads.
// D: the type of b (T, or of RESIDUAL's delta also float).
template <typename T, typename D, int OP, bool QUANT, bool ALIGNED, int E, bool WARP_ROW, bool WHOLE, int MAX_THREADS, int BLOCKS>
__global__ void __launch_bounds__(MAX_THREADS, BLOCKS) rows_kernel(const Args p) {
  using Rw = Raw<T, ALIGNED>;
  constexpr bool PAIRS = ALIGNED || sizeof(D) == 2;
  __shared__ float2 red[2][32];
  griddep_launch_dependents();
  griddep_wait();
  const long long row = WARP_ROW ? blockIdx.x * 4ll + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP_ROW && row >= p.n_rows) return;
  const int n = p.n;
  const int t = WARP_ROW ? threadIdx.x & 31 : threadIdx.x, per_octet = 8 * (WARP_ROW ? 32 : blockDim.x), per_chunk = E * per_octet;
  const T* a = static_cast<const T*>(p.a) + row * p.lda;
  const D* b = static_cast<const D*>(p.b) + row * p.ldb;
  const T* weight = static_cast<const T*>(p.weight);
  const T* post = static_cast<const T*>(p.post_weight);
  const T* gate = static_cast<const T*>(p.gate);
  if (OP == RESIDUAL && gate) gate += row / p.rows_per_gate * n;
  T* hidden = static_cast<T*>(p.hidden_out) + row * n;
  // the first octet begins where the row that is written lies on 16 bytes
  int i0 = t * 8;
  if (!ALIGNED && OP == RESIDUAL) i0 -= static_cast<int>((reinterpret_cast<uintptr_t>(hidden) & 15) / sizeof(T));
  constexpr bool NORMED = OP == RESIDUAL || OP == NORM_ROWS;
  const auto inside = [&](int i) { return ALIGNED ? i < n : i < n && i + 8 > 0; };
  const auto factors = [&](const T* src, int i, float(&f)[8]) {
    Rw w;
    w.load(src, i, n);
    w.octet(src, i, n).get(f);
  };

  Octet<T> x[E];                                     // RESIDUAL: hidden
  Octet<D> y[E];                                     // delta
  // all loads of a chunk on their way, then the values
  const auto fetch = [&](const T* src_x, const D* src_y, int c0) {
    Rw rx[E];
    Raw<D, ALIGNED> ry[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = i0 + c0 + e * per_octet;
      if (inside(i)) {
        if (src_x) rx[e].load(src_x, i, n);
        if (src_y) ry[e].load(src_y, i, n);
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = i0 + c0 + e * per_octet;
      if (inside(i)) {
        if (src_x) x[e] = rx[e].octet(src_x, i, n);
        if (src_y) y[e] = ry[e].octet(src_y, i, n);
      }
    }
  };
  if (WHOLE) fetch(a, OP == RESIDUAL || OP == SILU_MUL ? b : nullptr, 0);

  float rd = 1.0f;                                   // RESIDUAL: 1 / rms of delta
  if (OP == RESIDUAL && post) {
    Squares squares;
    for (int c0 = 0; c0 < (WHOLE ? 1 : n + 8); c0 += per_chunk) {
      if (!WHOLE) fetch(nullptr, b, c0);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (!inside(i0 + c0 + e * per_octet)) continue;
        float v[8];
        y[e].get(v);
        squares.template add<PAIRS>(v);
      }
      if (!WHOLE) squares.template end_chunk<PAIRS>();
    }
    float ss = squares.template total<PAIRS, WHOLE>();
    reduce_row<WARP_ROW>(ss, red[0]);
    rd = rsqrtf(ss / static_cast<float>(n) + p.eps);
  }

  Squares squares;
  float amax = 0.0f;
  constexpr bool KEEP = WHOLE && QUANT && (OP == SILU_MUL || (OP != ROWS && PAIRS && E <= 4));
  float value[KEEP ? E : 1][8];                      // what is quantised (of NORMED rows without the factor rr)
  for (int c0 = 0; c0 < (WHOLE ? 1 : n + 8); c0 += per_chunk) {
    if (!WHOLE) fetch(a, OP == RESIDUAL || OP == SILU_MUL ? b : nullptr, c0);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = i0 + c0 + e * per_octet;
      if (!inside(i)) continue;
      float v[8], u[8];
      x[e].get(v);
      const auto magnitudes = [&](const float(&m)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(m[j]));
        if constexpr (KEEP) {
#pragma unroll
          for (int j = 0; j < 8; ++j) value[e][j] = m[j];
        }
      };
      if constexpr (OP == SILU_MUL) {
        y[e].get(u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = silu_mul(v[j], u[j]);
        magnitudes(v);
        continue;
      }
      if (OP == RESIDUAL) {
        float f[8];
        y[e].get(u);
        if (post) {
          factors(post, i, f);
          scale8<PAIRS>(u, rd);
          mul8<PAIRS>(u, f);
        }
        if (gate) {
          factors(gate, i, f);
          mul8<PAIRS>(u, f);
        }
        add_scaled8<PAIRS>(v, p.scale, u);
        x[e].set(v);                                 // the value that is stored, which the norm reads
        x[e].template store<ALIGNED>(hidden, i, n);
        x[e].get(v);
      }
      if (NORMED) {
        squares.template add<PAIRS>(v);
        if (QUANT) {
          factors(weight, i, u);
          mul8<PAIRS>(v, u);
          magnitudes(v);
        }
      } else {
        magnitudes(v);
      }
    }
    if (!WHOLE && NORMED) squares.template end_chunk<PAIRS>();
  }
  if (!QUANT && !weight) return;                     // RESIDUAL without a norm after it
  float ss = squares.template total<PAIRS, WHOLE>();
  reduce_row<WARP_ROW>(ss, amax, red[1]);
  const float rr = NORMED ? rsqrtf(ss / static_cast<float>(n) + p.eps) : 1.0f;
  const bool finite = amax < __uint_as_float(0x7F800000u);       // (false for NaN)
  // the row's scale, without the factor rr
  const float s = amax == 0.0f ? 1.0f : fmaxf(__fdiv_rn(amax, 127.0f), 1.17549435e-38f);
  const float inv = NORMED && amax > 1e-30f ? __fdiv_rn(127.0f, amax) : __fdiv_rn(1.0f, s);
  if (QUANT && t == 0) p.scales[row] = !finite ? __uint_as_float(0x7FC00000u) : amax == 0.0f ? 1.0f : NORMED ? s * rr : s;

  for (int c0 = 0; c0 < (WHOLE ? 1 : n + 8); c0 += per_chunk) {
    if (!WHOLE) fetch(OP == RESIDUAL ? hidden : a, OP == SILU_MUL ? b : nullptr, c0);        // (hidden: each thread reads what it has written itself)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = i0 + c0 + e * per_octet;
      if (!inside(i)) continue;
      float v[8], u[8];
      if constexpr (KEEP) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = value[e][j];
      } else {
        x[e].get(v);
        if (OP == SILU_MUL) {
          y[e].get(u);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = silu_mul(v[j], u[j]);
        } else if (NORMED) {
          factors(weight, i, u);
          if (!QUANT) scale8<PAIRS>(v, rr);
          mul8<PAIRS>(v, u);
        }
      }
      if (QUANT) {
        store_q<ALIGNED, OP == ROWS, NORMED && sizeof(T) == 2>(static_cast<int8_t*>(p.out) + row * p.ldo, i, n, v, s, inv, finite);
      } else {
        Octet<T> o;
        o.set(v);
        o.template store<ALIGNED>(static_cast<T*>(p.out) + row * p.ldo, i, n);
      }
    }
  }
}

// ---------------------------------------------------------------------------- host side
template <typename T, typename D, int OP, bool QUANT, bool ALIGNED, int E, bool WARP_ROW, bool WHOLE, int MAX_THREADS, int BLOCKS>
int launch_form(const Args& p, int threads, cudaStream_t st) {
  const long long blocks = WARP_ROW ? (p.n_rows + 3) / 4 : p.n_rows;
  if (blocks > 2147483647LL) { set_error("more than 2^31 rows"); return LCQ_ERR_UNSUPPORTED; }
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[1];
  glue::pdl_config(cfg, attr, dim3(static_cast<unsigned>(blocks)), dim3(threads), st);
  LCQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, rows_kernel<T, D, OP, QUANT, ALIGNED, E, WARP_ROW, WHOLE, MAX_THREADS, BLOCKS>, p));
  return LCQ_OK;
}
// The forms and where each is the faster (us, B200; n values a row, E octets a thread).
//   a warp a row, four rows a block   n <= 512 (20,000 x 512 quantised: 8.1, 21.3 with a block a row, whose launches bound it), and <= 1024 with one operand
//   E = 1, most threads a row         few rows, where latency counts (1 x 4096: 2.6; E = 2 3.2, E = 4 4.4), and RESIDUAL up to 2048 values or 8 Mi in all
//   E = 4, most bytes on their way    all other 16-bit rows up to 16,384 (8192 x 8192 RESIDUAL: 87; E = 1 122, E = 2 98, E = 8 101)
//   E = 2                             float32, and rows off 16 bytes, which hold more registers for each octet (4000 x 5003: 48; E = 1 59, E = 4 56)
//                                     (a float32 delta beside 16 bits counts as float32: 1000 x 2048 4.6 for 4.2 with 16 bits, 8192 x 8192 107 for 81, both at
//                                     the copy rate)
//   E = 8                             16-bit rows up to 32,768 of one operand (4000 x 28,672 quantised: 69; E = 4 93); of two, E = 4 in twice the threads
//                                     (1000 x 28,672 SILU_MUL: 39; E = 8 44, in chunks 58)
//   in chunks, E = 2                  longer rows, two blocks an SM (1000 x 50,001 bfloat16 SILU_MUL 150, one block 156; 1000 x 50,000 RESIDUAL 100 and 141); one for two
//                                     operands in float32, which do not fit into 64 registers (1000 x 50,000 RESIDUAL 206, two blocks 303; 64 x 20,001 14 and 30)
template <typename T, typename D, int OP, bool QUANT, bool ALIGNED>
int launch_aligned(const Args& p, int sm_count, cudaStream_t st) {
  constexpr bool HALF = sizeof(D) == 2, ONE = OP == ROWS || OP == NORM_ROWS;
  const int span = p.n + (ALIGNED ? 0 : 7);          // (an octet may begin up to seven values before the row)
  const auto threads = [&](int e) { return ((span + 8 * e - 1) / (8 * e) + 31) / 32 * 32; };
  const bool few = p.n_rows <= 2ll * sm_count;
  if (span <= 512 && p.n_rows >= 4) return launch_form<T, D, OP, QUANT, ALIGNED, 2, true, true, 128, 8>(p, 128, st);
  if constexpr (ONE) {
    if (span <= 1024 && !few) return launch_form<T, D, OP, QUANT, ALIGNED, 4, true, true, 128, 4>(p, 128, st);
  }
  if (span <= 8192 && (few || (HALF && ALIGNED && OP == RESIDUAL && (p.n <= 2048 || p.n_rows * p.n <= (8ll << 20)))))
    return launch_form<T, D, OP, QUANT, ALIGNED, 1, false, true, 1024, 2>(p, threads(1), st);
  if constexpr (!HALF || !ALIGNED) {
    if (span <= 8192) return launch_form<T, D, OP, QUANT, ALIGNED, 2, false, true, 512, 2>(p, threads(2), st);
    if (span <= 16384) return launch_form<T, D, OP, QUANT, ALIGNED, 4, false, true, 512, 1>(p, threads(4), st);
  } else {
    if (span <= 16384) return launch_form<T, D, OP, QUANT, ALIGNED, 4, false, true, 512, ONE ? 3 : 2>(p, threads(4), st);
  }
  if constexpr (HALF) {
    if constexpr (ONE) {
      if (span <= 32768) return launch_form<T, D, OP, QUANT, ALIGNED, 8, false, true, 512, 2>(p, threads(8), st);
    } else {
      if (span <= 32768) return launch_form<T, D, OP, QUANT, ALIGNED, 4, false, true, 1024, 1>(p, threads(4), st);
    }
  }
  return launch_form<T, D, OP, QUANT, ALIGNED, 2, false, false, 512, HALF || ONE ? 2 : 1>(p, 512, st);
}

// Octets as they lie where every row of every operand starts on 16 bytes (of q: on 8) and holds whole ones.
template <typename T, int OP, bool QUANT, typename D = T>
int launch(const Args& p, int sm_count, cudaStream_t st) {
  const auto rows_on_16 = [&](const void* q, long long ld) { return aligned(q, 16) && (ld * sizeof(T)) % 16 == 0; };
  const bool on_16 = p.n % 8 == 0 && rows_on_16(p.a, p.lda) && aligned(p.b, 16) && (p.ldb * sizeof(D)) % 16 == 0 && aligned(p.weight, 16) && aligned(p.post_weight, 16) &&
                     aligned(p.gate, 16) && aligned(p.hidden_out, 16) &&
                     (QUANT ? aligned(p.out, 8) && p.ldo % 8 == 0 : rows_on_16(p.out, p.ldo));
  return on_16 ? launch_aligned<T, D, OP, QUANT, true>(p, sm_count, st) : launch_aligned<T, D, OP, QUANT, false>(p, sm_count, st);
}

}  // namespace rows
}  // namespace lcq
