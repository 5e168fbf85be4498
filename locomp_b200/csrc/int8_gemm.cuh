// Int8 matrix product with a scale for each token and each output channel, on 5th-generation tensor cores.
//
//   out[m, n] = (sum_k x[m, k] * w[n, k]) * x_scales[m] * w_scales[n]
//
// The sum is exact: int32 (K at most 131,071, so that K * 128 * 128 fits), in whatever order its parts meet.  It is
// converted to float32 (rounded once), multiplied by the two scales in float32, and rounded to the output's type.
//
// Orientation: the MMA's M dimension is the weight row n, its N dimension the token m, for one token as for thousands.
// A team -- one CTA (CG = 1) or the two CTAs of a cluster (CG = 2) -- owns D[128 * CG n x bm m]; CTA r holds the weight
// rows 128 r .. 128 r + 127 and 1 / CG of the tokens.  Both operands go by TMA into stages of 128 k (one swizzled row of
// 128 bytes each) and are read from there by tcgen05.mma kind::i8; accumulators are int32 in tensor memory, two of them,
// so that the epilogue of one tile runs under the MMAs of the next.  With few tokens the tensor cores idle and the ring
// of stages does nothing but stream weights.
// A lane of the accumulator is a channel: its scale is one register, and a warp stores 32 consecutive channels of a token.
//
// Split of the work: whole tiles in turn while they fill all teams, the rest in pieces of fewer tokens; or, where there are few tiles, a
// cluster of CTAs shares the K of each tile and adds up over distributed shared memory.  (Cutting the last tiles along K between CTAs that meet
// through scratch was faster for 4 problems of 75, by 3 %, and made every call need scratch.)
//
// The weights' first stages are fetched into L2 while the kernel before this one still runs.  L2 is where all SMs' stores
// meet, so this is right whoever writes the weights; everything is read after that kernel has completed.
//
// Operands whose rows do not start on 16 bytes (K % 16 != 0 in contiguous storage, or an odd offset) have no tensor map.  They are first copied
// into rows that do, the weights 48 MiB at a time, so that the copy is multiplied out of L2.  (Loader warps that shifted the bytes on their way into
// the ring took two to four times as long: 333 x 4104 -> 5003 93 us, 1 x 577 -> 49152 28.6 us.)
//
// Every mbarrier wait is bounded; on expiry the kernel records a status code and unwinds.
#pragma once
#include "gemm_tc.cuh"

namespace lcq {
namespace int8_gemm {

using gemm_tc::Ring;
using gemm_tc::arrive_leader;
using gemm_tc::cluster_barrier;
using gemm_tc::leader_addr;
using gemm_tc::peer_addr;
using gemm_tc::store_remote;
using gemm_tc::tc_fence_after;
using gemm_tc::tc_fence_before;
using gemm_tc::tma_load_2d_pair;
using gemm_tc::tmem_alloc;
using gemm_tc::tmem_dealloc;
using gemm_tc::tmem_ld16;
using gemm_tc::tmem_ld32;
using gemm_tc::tmem_wait_ld;
using gemm_tc::umma_commit;
using gemm_tc::wait_bar;
using gemm_tc::warp_wait;

constexpr int BN = 128;                      // weight rows per CTA
constexpr int BK = 128;                      // k per stage: one swizzled row of 128 bytes, four MMAs
constexpr int W_STAGE = BN * BK;
constexpr int MAX_STAGES = 12;
// Warps 0 .. 7: two epilogue groups of four, which take the chunks of a tile's columns in turn (1024 x 16384 outputs of 1024 k: 31.9 us with one group,
// 23.1 with two; a third and a fourth changed nothing, nor did two chunks a trip to tensor memory).
constexpr int N_EPI = 8, WARP_TMA = 8, WARP_MMA = 9, NTHREADS = (WARP_MMA + 1) * 32;
constexpr int BAR_ALL = 1, BAR_GROUP = 2;    // named barriers: both groups; group g: BAR_GROUP + g
constexpr int MAX_K = 131071;
constexpr int MAX_SPLIT = 8;                 // CTAs of a cluster that share a tile's K

// Division of 0 <= n < 2^31 by a divisor of the host's choosing, as a product with its reciprocal (Granlund and Montgomery, Division by Invariant Integers
// using Multiplication, 1994): the walk's divisions by Params took 2000 clocks a tile.
struct Divisor {
  uint32_t mul;
  int shift;
  __host__ __device__ int divide(int n) const { return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul) >> shift); }
};
inline Divisor make_divisor(int d) {           // mul = ceil(2^(31 + l) / d), l = ceil(log2 d): exact for n < 2^31
  int l = 0;
  while ((1ll << l) < d) ++l;
  const uint64_t two = 1ull << (31 + l);
  return {static_cast<uint32_t>((two + static_cast<uint64_t>(d) - 1) / static_cast<uint64_t>(d)), 31 + l};
}

struct Params {
  void* out;                 // [M, N], rows ldo apart
  const float* x_scales;     // [M]
  const void* w_scales;      // [N]
  long long ldo;
  int M, N, K, w_scale_dtype;
  int bm;                    // tokens per tile (MMA N): a multiple of 16 CG, at most 256
  int piece_bm;              // bm / tail
  int tn, tm, n_tiles;
  int group;                 // token tiles that are walked together
  int nst;                   // 128-k stages per tile
  int teams;                 // CTAs (CG = 1) or pairs (CG = 2) launched
  int full, tail;            // tiles full .. are cut into `tail` pieces of bm / tail tokens (a last wave that would be mostly empty)
  int split;                 // > 1: a cluster of `split` CTAs per tile, each with its share of K
  int depth;                 // stages in the ring
  int tmem_cols;
  int vec;                   // whether rows of out start on 16 bytes
  Divisor by_group_tiles, by_group, by_last_group, by_tail;     // (tn * group tiles a group; token tiles in a group and in the last one)
};

// The segments of one team: (tile or piece of one, stages st0 .. st1 - 1).  Every role walks them in the same order.
struct Walk {
  int item, step;            // tiles, then pieces; how far apart a team's are
  int tile, st0, st1;
  int mt, nt;                // the tile's place
  int m0, bm;                // first token and their number
  __host__ __device__ Walk(const Params& p, int team) {
    if (p.split > 1) {
      item = team / p.split;
      const int r = team - item * p.split;
      st0 = p.nst * r / p.split;
      st1 = p.nst * (r + 1) / p.split;
      step = p.n_tiles;
    } else {
      item = team;
      st0 = 0;
      st1 = p.nst;
      step = p.teams;
    }
  }
  __host__ __device__ bool next(const Params& p) {
    for (;;) {
      tile = item;
      int piece = 0;
      bm = p.bm;
      if (item >= p.full) {
        const int i = item - p.full, of = p.by_tail.divide(i);
        tile = p.full + of;
        piece = i - of * p.tail;
        bm = p.piece_bm;
      }
      if (tile >= p.n_tiles) return false;
      item += step;
      // `group` token tiles at a time against all channels, tokens first: what runs at the same time shares its operands in L2
      const int g = p.by_group_tiles.divide(tile), in = tile - g * p.group * p.tn;
      const bool last = p.tm - g * p.group < p.group;
      const int rows = last ? p.tm - g * p.group : p.group;
      nt = last ? p.by_last_group.divide(in) : p.by_group.divide(in);
      mt = g * p.group + in - nt * rows;
      m0 = mt * p.bm + piece * bm;
      if (m0 < p.M) return true;               // (a piece past the last token is no work)
    }
  }
};

enum { FLAG_ABORT, ISSUED_0, ISSUED_1, N_FLAGS };
struct Smem { int out, xs, bars, tmem_slot, flags, total; };   // offsets from the 1024-byte aligned base; the ring comes first
__host__ __device__ inline int stage_bytes(int bm, int cg) { return W_STAGE + (bm / cg) * BK; }
// Tiles of 16 tokens are stored from registers, higher ones through shared memory (two buffers of 8 KB for each group).
__host__ __device__ inline bool staged(int bm) { return bm > 16; }
constexpr int OUT_BUFFER = 8192;
constexpr int OUT_BOX = 16;                  // tokens of a copy out of it: tiles are multiples of 16, so none reaches into the next tile
__host__ __device__ inline Smem smem_map(int bm, int cg, int depth) {
  Smem s;
  s.out = depth * stage_bytes(bm, cg);
  s.xs = s.out + (staged(bm) ? 4 * OUT_BUFFER : 0);         // scales of a tile's tokens; two tiles in turn
  s.bars = s.xs + (staged(bm) ? 2 * 256 * 4 : 0);
  s.tmem_slot = s.bars + (2 * MAX_STAGES + 5) * 8;          // full, empty [MAX_STAGES]; full_d, empty_d [2]; drained
  s.flags = s.tmem_slot + 8;
  s.total = s.flags + 4 * N_FLAGS;
  return s;
}

// kind::i8 instruction descriptor: D = s32, A = B = s8, both K-major, M = 128 * CG, N = bm.
__host__ __device__ inline uint32_t make_idesc(int bm, int cg) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(bm >> 3) << 17) | (static_cast<uint32_t>((BN * cg) >> 4) << 24);
}
// D[tmem] (+)= A[smem] * B[smem] over a stage of 128 k: four MMAs, issued by one elected lane of a whole warp.
// a, b: the low words of the descriptors (their high words are alike).
#define LCQ_I8_MMA(CG, P) "tcgen05.mma.cta_group::" #CG ".kind::i8 [%0], ad, bd, %3, " P ";\n\t"
#define LCQ_I8_NEXT "add.u32 a, a, 2;\n\tadd.u32 b, b, 2;\n\tmov.b64 ad, {a, %5};\n\tmov.b64 bd, {b, %5};\n\t"
#define LCQ_I8_STAGE(CG)                                                                                            \
  asm volatile(                                                                                                     \
      "{\n\t.reg .pred p, q, e;\n\t.reg .b64 ad, bd;\n\t.reg .b32 a, b;\n\t"                                        \
      "elect.sync _|e, 0xffffffff;\n\t@!e bra ISSUED;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t"         \
      "mov.b32 a, %1;\n\tmov.b32 b, %2;\n\tmov.b64 ad, {a, %5};\n\tmov.b64 bd, {b, %5};\n\t"                        \
      LCQ_I8_MMA(CG, "p") LCQ_I8_NEXT LCQ_I8_MMA(CG, "q") LCQ_I8_NEXT LCQ_I8_MMA(CG, "q") LCQ_I8_NEXT               \
      LCQ_I8_MMA(CG, "q") "ISSUED:\n\t}"                                                                            \
      ::"r"(d_tmem), "r"(a), "r"(b), "r"(idesc), "r"(first), "n"(gemm_tc::B_DESC_HI) : "memory")
template <int CG>
__device__ __forceinline__ void mma_stage(uint32_t d_tmem, uint32_t a, uint32_t b, uint32_t idesc, uint32_t first) {
  if (CG == 2) LCQ_I8_STAGE(2);
  else LCQ_I8_STAGE(1);
}
#undef LCQ_I8_STAGE
#undef LCQ_I8_NEXT
#undef LCQ_I8_MMA

__device__ __forceinline__ void tma_prefetch_2d(const void* tmap, int x, int y) {      // into L2 only
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(tmap), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ float load_scale(const void* s, long long i, int dtype) {
  return dtype == LCQ_F32 ? static_cast<const float*>(s)[i]
         : dtype == LCQ_F16 ? __half2float(static_cast<const __half*>(s)[i])
                            : __bfloat162float(static_cast<const __nv_bfloat16*>(s)[i]);
}

// After a wait ran out in the CTA or its partner: waits for what they still have under way (the MMAs, and the copies into the last
// stages, which nobody waits for any more).  A CTA of a pair may have loaded its part of a stage whose other part was
// never issued: the barrier is then given the missing part, or armed for the one that comes.  All threads; in a pair between two
// cluster barriers.
template <int CG>
__device__ __noinline__ void drain(const Params& p, uint8_t* smem, int team, uint32_t crank) {
  const Smem L = smem_map(p.bm, CG, p.depth);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.bars);
  uint64_t* drained = full + 2 * MAX_STAGES + 4;
  const volatile int* flags = reinterpret_cast<const volatile int*>(smem + L.flags);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (warp == WARP_MMA) {
    if (crank == 0) umma_commit<CG>(drained);
    __syncwarp();
    mbar_wait_landed(drained, 0);
  } else if (warp == WARP_TMA && lane == 0 && crank == 0) {
    const int mine = flags[ISSUED_0], other = CG == 2 ? flags[ISSUED_1] : mine, n = mine > other ? mine : other;
    int i = 0;
    for (Walk w(p, team); i < n && w.next(p);) {
      for (int st = w.st0; st < w.st1 && i < n; ++st, ++i) {
        if (i < n - p.depth) continue;
        const int bytes = stage_bytes(w.bm, CG);
        uint64_t* bar = full + i % p.depth;
        if (i >= mine) mbar_expect_tx(bar, bytes);
        else if (i >= other) asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
        mbar_wait_landed(bar, (i / p.depth) & 1);
      }
    }
  }
  __syncthreads();
}

// A chunk of columns (tokens) of a tile, as the epilogue takes them: 8 KB of output.
template <typename OT> __host__ __device__ constexpr int chunk_columns() { return sizeof(OT) == 2 ? 32 : 16; }
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&v)[32]) { tmem_ld32(taddr, v); }
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&v)[16]) { tmem_ld16(taddr, v); }
__device__ __forceinline__ float scaled(uint32_t sum, float xs, float ws) { return static_cast<float>(static_cast<int>(sum)) * xs * ws; }

// Stores a chunk from registers: 32 channels of a token at a time.
template <typename OT, int C>
__device__ __forceinline__ void store_direct(const uint32_t (&v)[C], OT* out, long long ldo, bool there, int columns, const float* x_scales, float ws, int lane) {
  const float xs = lane < columns ? x_scales[lane] : 0.0f;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const float s = __shfl_sync(0xffffffffu, xs, i);
    if (there && i < columns) *out = from_f32<OT>(scaled(v[i], s, ws));
    out += ldo;
  }
}

__device__ __forceinline__ void put2(float* p, float* q, float2 v) { *p = v.x; *q = v.y; }
__device__ __forceinline__ void put2(__half* p, __half* q, float2 v) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  *p = __low2half(h);
  *q = __high2half(h);
}
__device__ __forceinline__ void put2(__nv_bfloat16* p, __nv_bfloat16* q, float2 v) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  *p = __low2bfloat16(h);
  *q = __high2bfloat16(h);
}

// Where rows of out do not start on 16 bytes, a row's 128 channels lie rotated in shared memory, by the place of its first one in its 16 bytes of global
// memory: so that sixteen bytes are sixteen bytes on both sides.  Tiles begin at multiples of 16 tokens and 128 channels, so a row's rotation goes by its
// number in the chunk alone.  (A thread finds its places once and its whole pieces' rows share one rotation.  Found for each value, and with the rows' ends
// among the pieces: 1074 x 383 -> 31476 in bf16 68 us, now 48; 2048 x 512 -> 5003 26.6 and 26.6 in float32, now 18.5 and 21; aligned outputs take the same.)
template <typename OT> struct Rotation {
  static constexpr int EACH = 16 / static_cast<int>(sizeof(OT));         // values in 16 bytes
  int first, step;                             // of a chunk's first token; from token to token
  __device__ __forceinline__ Rotation(const void* out, long long ldo)
      : first(static_cast<int>(reinterpret_cast<uintptr_t>(out) / sizeof(OT) & (EACH - 1))), step(static_cast<int>(ldo & (EACH - 1))) {}
  __device__ __forceinline__ int of(int row) const { return (first + row * step) & (EACH - 1); }
};
// A chunk into shared memory, [token][128 channels], row i's channel of this lane at place[i % EACH]: from there 256 (512) consecutive bytes of a token go
// out together.  (Stored from registers, 64 or 128 bytes a warp, a 1024 x 16384 output took 56 us in 16 bits and 32 us in float32, whatever K.)
template <typename OT, int C>
__device__ __forceinline__ void stage_chunk(const uint32_t (&v)[C], OT* buf, const int (&place)[Rotation<OT>::EACH], const float* xs, uint64_t ws2) {
#pragma unroll
  for (int i = 0; i < C; i += 4) {
    const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(xs + i);
#pragma unroll
    for (int j = i; j < i + 4; j += 2) {
      const uint64_t sum = pack_pair(static_cast<float>(static_cast<int>(v[j])), static_cast<float>(static_cast<int>(v[j + 1])));
      put2(buf + j * BN + place[j % Rotation<OT>::EACH], buf + (j + 1) * BN + place[(j + 1) % Rotation<OT>::EACH],
           unpack_pair(mul_pair(mul_pair(sum, j == i ? s.x : s.y), ws2)));
    }
  }
}
// A chunk's rotated rows from shared memory to global, by a group's 128 threads: 16 bytes a thread; then the pieces that hold a row's last and first channels,
// and those that the last channel of all cuts, value by value.
template <typename OT, int C>
__device__ __forceinline__ void store_rotated(const OT* buf, OT* out, long long ldo, Rotation<OT> rot, int channels, int columns, int t) {
  constexpr int EACH = Rotation<OT>::EACH, PIECES = BN / EACH;
  {
    const int piece = t % PIECES, shift = rot.of(t / PIECES), c0 = piece * EACH - shift;       // (the rows of a thread are multiples of EACH apart)
    if (c0 >= 0 && c0 + EACH <= channels) {
#pragma unroll
      for (int i = 0; i < C * PIECES / 128; ++i) {
        const int row = i * (128 / PIECES) + t / PIECES;
        if (row < columns) *reinterpret_cast<uint4*>(out + row * ldo + c0) = *reinterpret_cast<const uint4*>(buf + row * BN + piece * EACH);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < (C * EACH + 127) / 128; ++i) {
    const int row = i * (128 / EACH) + t / EACH, shift = rot.of(row), c = (t % EACH - shift) & (BN - 1);
    if (shift != 0 && row < columns && c < channels) out[row * ldo + c] = buf[row * BN + t % EACH];
  }
  if (channels < BN) {                         // the tile's last channels
    for (int row = t / 32; row < columns; row += 4) {
      const int shift = rot.of(row), from = channels - (channels + shift) % EACH;              // the first one that no whole piece holds
      const int c = from + t % 32;
      if (c < channels && c >= 0) out[row * ldo + c] = buf[row * BN + ((c + shift) & (BN - 1))];
    }
  }
}
// A box of out from shared memory; what lies past its last row or column is left out.
__device__ __forceinline__ void tma_store_2d(const void* tmap, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];\n\t"
               "cp.async.bulk.commit_group;"
               ::"l"(tmap), "r"(smem_u32(src)), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tma_stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ bool all_epilogue_warps(bool ok) {
  uint32_t all;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all) : "r"(ok ? 1u : 0u), "n"(BAR_ALL), "n"(N_EPI * 32) : "memory");
  return all != 0;
}

template <int CG, typename OT>
__global__ void __launch_bounds__(NTHREADS, 1)
int8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_piece, const __grid_constant__ CUtensorMap tmap_w,
                 const __grid_constant__ CUtensorMap tmap_out, const __grid_constant__ Params p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  const Smem L = smem_map(p.bm, CG, p.depth);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.bars);
  uint64_t* empty = full + MAX_STAGES;
  uint64_t* full_d = empty + MAX_STAGES;
  uint64_t* empty_d = full_d + 2;
  uint64_t* drained = empty_d + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L.tmem_slot);
  volatile int* flag_abort = reinterpret_cast<volatile int*>(smem + L.flags);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const uint32_t crank = CG == 2 ? blockIdx.x & 1 : 0;
  const int team = blockIdx.x / CG;
  const int stage = stage_bytes(p.bm, CG);

  if (threadIdx.x == 0) {
    // full and empty_d are used in the pair's first CTA only; commits arrive in both
    for (int i = 0; i < MAX_STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&full_d[i], 1); mbar_init(&empty_d[i], N_EPI * CG); }
    mbar_init(drained, 1);
    *flag_abort = 0;
    fence_barrier_init();
  }
  if (warp == WARP_TMA && lane == 0) {
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
    int ahead = p.depth;
    for (Walk w(p, team); ahead > 0 && w.next(p);) {
      for (int st = w.st0; st < w.st1 && ahead > 0; ++st, --ahead)
        tma_prefetch_2d(&tmap_w, st * BK, w.nt * (CG * BN) + static_cast<int>(crank) * BN);
    }
  }
  if (warp == WARP_MMA) tmem_alloc<CG>(tmem_slot, p.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (CG == 2) cluster_barrier();             // the other CTA's barriers exist
  if (threadIdx.x == 0) griddep_launch_dependents();       // after tmem_alloc: see gemm_tc.cuh
  const uint32_t tmem_base = *tmem_slot;

#define LCQ_GIVE_UP(code)                                                                              \
  do {                                                                                                 \
    *flag_abort = 1;                                                                                   \
    if (CG == 2) store_remote(peer_addr(smem_u32(smem + L.flags + 4 * FLAG_ABORT), crank ^ 1u), 1);    \
    atomicExch(&g_device_status, (code));                                                              \
  } while (0)

  if (warp == WARP_TMA) {
    // ------------------------------------------------------------ this CTA's weight rows and tokens of each stage
    if (lane == 0) {
      griddep_wait();
      Ring r = {0, 0};
      bool ok = true;
      int issued = 0;
      for (Walk w(p, team); ok && w.next(p);) {
        const int n0 = w.nt * (CG * BN) + static_cast<int>(crank) * BN, m0 = w.m0 + static_cast<int>(crank) * (w.bm / CG);
        const int bytes = stage_bytes(w.bm, CG);
        const CUtensorMap* tmap = w.bm == p.bm ? &tmap_x : &tmap_piece;
        for (int st = w.st0; st < w.st1; ++st, r.step(p.depth)) {
          if (!wait_bar(flag_abort, &empty[r.i], r.phase ^ 1u)) { LCQ_GIVE_UP(60); ok = false; break; }
          uint8_t* dst = smem + r.i * stage;
          if (crank == 0) mbar_expect_tx(&full[r.i], CG * bytes);
          if (CG == 2) {
            const uint32_t bar = leader_addr<CG>(full + r.i);
            tma_load_2d_pair(dst, &tmap_w, bar, st * BK, n0);
            tma_load_2d_pair(dst + W_STAGE, tmap, bar, st * BK, m0);
          } else {
            tma_load_2d(dst, &tmap_w, full + r.i, st * BK, n0);
            tma_load_2d(dst + W_STAGE, tmap, full + r.i, st * BK, m0);
          }
          ++issued;
        }
      }
      if (CG == 2) store_remote(peer_addr(smem_u32(smem + L.flags + 4 * (ISSUED_0 + crank)), 0), issued);
      else flag_abort[ISSUED_0] = issued;
    }
  } else if (warp == WARP_MMA) {
    // ------------------------------------------------------------ MMA issuer: one warp for the team
    griddep_wait();                            // (so that the limits of its waits count this kernel's time alone)
    if (crank == 0) {
      const uint32_t desc0 = gemm_tc::make_b_desc(smem_u32(smem));             // descriptors count 16-byte units
      Ring r = {0, 0}, rd = {0, 0};
      bool ok = true;
      for (Walk w(p, team); ok && w.next(p); rd.step(2)) {
        if (!warp_wait(flag_abort, &empty_d[rd.i], rd.phase ^ 1u)) { if (lane == 0) LCQ_GIVE_UP(61); ok = false; break; }
        tc_fence_after();
        const uint32_t d_t = tmem_base + rd.i * p.bm, idesc = make_idesc(w.bm, CG);
        for (int st = w.st0; st < w.st1; ++st, r.step(p.depth)) {
          if (!warp_wait(flag_abort, &full[r.i], r.phase)) { if (lane == 0) LCQ_GIVE_UP(62); ok = false; break; }
          tc_fence_after();
          const uint32_t a = desc0 + r.i * static_cast<uint32_t>(stage >> 4);
          mma_stage<CG>(d_t, a, a + (W_STAGE >> 4), idesc, st != w.st0);
          umma_commit<CG>(&empty[r.i]);
        }
        if (ok) umma_commit<CG>(&full_d[rd.i]);
      }
    }
  } else if (warp < N_EPI) {
    // ------------------------------------------------------------ epilogue warps: TMEM -> global
    griddep_wait();                            // out may still be in the preceding kernel's use
    constexpr int C = chunk_columns<OT>();
    const int group = warp >> 2, in_group = warp & 3;
    const int r = in_group * 32 + lane;        // weight row of the tile = TMEM lane
    const uint32_t lane_taddr = tmem_base + (static_cast<uint32_t>(in_group * 32) << 16);
    const uint32_t empty_d0 = leader_addr<CG>(empty_d);
    const bool stage_out = staged(p.bm);
    float* xs_tile = reinterpret_cast<float*>(smem + L.xs);
    uint8_t* buffers = smem + L.out + group * 2 * OUT_BUFFER;
    int buffer = 0;
    const Rotation<OT> rot(p.out, p.ldo);      // (none where p.vec)
    int place[Rotation<OT>::EACH];
#pragma unroll
    for (int j = 0; j < Rotation<OT>::EACH; ++j) place[j] = (r + rot.of(j)) & (BN - 1);
    // The scales of a tile are on their way while the tile before it is stored: fetched in its own turn they showed in every short tile.
    Walk next(p, team);
    bool more = next.next(p);
    float ws_next = 0.0f, xs_next = 0.0f;
    const auto fetch_scales = [&] {
      const long long n = static_cast<long long>(next.nt) * (CG * BN) + static_cast<int>(crank) * BN + r;
      const long long m = static_cast<long long>(next.m0) + static_cast<int>(threadIdx.x);
      if (n < p.N) ws_next = load_scale(p.w_scales, n, p.w_scale_dtype);
      if (stage_out && static_cast<int>(threadIdx.x) < next.bm && m < p.M) xs_next = p.x_scales[m];
    };
    if (more) fetch_scales();
    Ring rd = {0, 0};
    for (; more; rd.step(2)) {
      const Walk w = next;
      const float ws = ws_next;
      const int n0 = w.nt * (CG * BN) + static_cast<int>(crank) * BN, n = n0 + r, m0 = w.m0;
      const bool there = n < p.N;
      const uint32_t d_t = lane_taddr + rd.i * p.bm;
      const int rows = p.M - m0 < w.bm ? p.M - m0 : w.bm;
      const float* xs = p.x_scales + m0;
      OT* out = static_cast<OT*>(p.out) + m0 * p.ldo + n0;
      if (stage_out) {
        xs_tile = reinterpret_cast<float*>(smem + L.xs) + rd.i * 256;    // (those of the tile before the last: read by all before the barrier of the last)
        if (static_cast<int>(threadIdx.x) < w.bm) xs_tile[threadIdx.x] = xs_next;
      }
      more = next.next(p);
      if (more) fetch_scales();
      if (!all_epilogue_warps(wait_bar(flag_abort, &full_d[rd.i], rd.phase))) { if (lane == 0) LCQ_GIVE_UP(63); break; }
      tc_fence_after();
      if (CG == 1 && p.split > 1) break;       // the cluster adds up its shares below
      for (int c0 = group * C; c0 < rows; c0 += 2 * C) {
        uint32_t v[C];
        tmem_load(d_t + c0, v);
        tmem_wait_ld();
        const int columns = rows - c0 < C ? rows - c0 : C;
        if (stage_out) {
          OT* buf = reinterpret_cast<OT*>(buffers + buffer * OUT_BUFFER);
          stage_chunk<OT, C>(v, buf, place, xs_tile + c0, pack_pair(ws, ws));
          if (p.vec) {
            fence_async_smem();                // the copy reads through the async proxy
            if (in_group == 0 && lane == 0) tma_stores_read();        // the copy before this one has left the other buffer, which comes next
            named_bar_sync(BAR_GROUP + group, 128);
            if (in_group == 0 && lane == 0 && n0 < p.N) {
              for (int h = 0; h < columns; h += OUT_BOX) tma_store_2d(&tmap_out, buf + h * BN, n0, m0 + c0 + h);
            }
          } else {
            named_bar_sync(BAR_GROUP + group, 128);
            store_rotated<OT, C>(buf, out + c0 * p.ldo, p.ldo, rot, p.N - n0 < BN ? p.N - n0 : BN, columns, r);
          }
          buffer ^= 1;
        } else {
          store_direct<OT, C>(v, out + r + c0 * p.ldo, p.ldo, there, columns, xs + c0, ws, lane);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_leader<CG>(empty_d0 + rd.i * 8);
    }
    if (in_group == 0 && lane == 0) tma_stores_read();      // the buffers outlive the copies
  }
#undef LCQ_GIVE_UP

  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_barrier();    // neither CTA leaves while the other may still arrive on its barriers or the pair's MMAs read its memory
  if (*flag_abort) {
    drain<CG>(p, smem, team, crank);
    if (CG == 2) cluster_barrier();
  }
  if (CG == 1 && p.split > 1) {
    // One tile per cluster, its K shared out: CTA d settles columns d * cw .. of the tile.  Every CTA sends each of the others its
    // part of their columns (into the ring, which nobody uses any more).
    Walk w(p, team);
    w.next(p);
    const int me = team % p.split, m0 = w.m0;
    const int rows = p.M - m0 < p.bm ? p.M - m0 : p.bm;
    const int cw = (rows + p.split - 1) / p.split;
    const int r = (warp & 3) * 32 + lane;
    cluster_barrier();
    if (warp < N_EPI) {
      tc_fence_after();
      const uint32_t mine = smem_u32(smem) + (me * cw * BN + r) * 4;
      for (int c0 = (warp >> 2) * 16; c0 < rows; c0 += 32) {
        uint32_t v[16];
        tmem_ld16(tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16) + c0, v);
        tmem_wait_ld();
        int d = c0 / cw, j = c0 - d * cw;
        uint32_t dst = peer_addr(mine + j * (BN * 4), d);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (c0 + i < rows) store_remote(dst, static_cast<int>(v[i]));
          dst += BN * 4;
          if (++j == cw && d + 1 < p.split) { j = 0; ++d; dst = peer_addr(mine, d); }
        }
      }
      tc_fence_before();
    }
    cluster_barrier();
    const int n = w.nt * BN + r;
    if (warp < N_EPI && n < p.N && *flag_abort == 0) {
      const int* got = reinterpret_cast<const int*>(smem) + r;
      const float ws = load_scale(p.w_scales, n, p.w_scale_dtype);
      OT* out = static_cast<OT*>(p.out) + (m0 + me * cw) * p.ldo + n;
      for (int j = warp >> 2; j < cw && me * cw + j < rows; j += 2) {
        int sum = 0;
        for (int q = 0; q < p.split; ++q) sum += got[(q * cw + j) * BN];
        out[j * p.ldo] = from_f32<OT>(static_cast<float>(sum) * p.x_scales[m0 + me * cw + j] * ws);
      }
    }
  }
  if (warp == WARP_MMA) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc<CG>(tmem_base, p.tmem_cols);
  }
}

// 16 bytes from any address: the two aligned pieces they lie in, and their bytes shifted into place.
struct Piece {
  uint4 a, b;
  int off;
  // The first `valid` bytes exist (at most 0: none).  Only aligned pieces that hold a byte that exists are read.
  __device__ __forceinline__ void load(const uint8_t* p, int valid) {
    off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
    const uint4* q = reinterpret_cast<const uint4*>(p - off);
    a = valid > 0 ? q[0] : make_uint4(0u, 0u, 0u, 0u);
    b = off + (valid < 16 ? valid : 16) > 16 ? q[1] : make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ uint4 get(int valid) const {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (off & 8) {
#pragma unroll
      for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (off & 4) {
#pragma unroll
      for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __funnelshift_r(w[i], w[i + 1], (off & 3) * 8);
    if (valid < 16) {                          // the end of a row: what follows reads as zero
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int left = valid - 4 * i;
        r[i] = left >= 4 ? r[i] : left <= 0 ? 0u : r[i] & ((1u << (8 * left)) - 1u);
      }
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
  }
};
// Rows of K bytes, ld apart, into rows of `per_row` pieces of 16 bytes (the last one filled up with zeros): of two operands, one after the other.
struct AlignJob {
  const uint8_t* src;
  long long ld;
  uint4* dst;
  int pieces;                // all in all
};
__global__ void __launch_bounds__(256) align_rows_kernel(const AlignJob first, const AlignJob second, int K, int per_row, Divisor by_per_row) {
  griddep_launch_dependents();
  griddep_wait();
  constexpr int EACH = 4;
  const long long stride = gridDim.x * 256ll, total = static_cast<long long>(first.pieces) + second.pieces;
  for (long long i0 = blockIdx.x * 256ll + threadIdx.x; i0 < total; i0 += EACH * stride) {
    Piece v[EACH];
    uint4* dst[EACH];
    int valid[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
      const long long i = i0 + j * stride;
      const AlignJob& job = i < first.pieces ? first : second;
      const int at = i < total ? static_cast<int>(i < first.pieces ? i : i - first.pieces) : 0;
      const int row = by_per_row.divide(at), k = (at - row * per_row) * 16;
      dst[j] = job.dst + at;
      valid[j] = i < total ? K - k : 0;
      v[j].load(job.src + row * job.ld + k, valid[j]);
    }
#pragma unroll
    for (int j = 0; j < EACH; ++j)
      if (i0 + j * stride < total) *dst[j] = v[j].get(valid[j]);
  }
}

// ---------------------------------------------------------------------------- host side
struct Tiling { int cg, bm, tn, tm, n_tiles, group, teams, full, tail, split, depth; };

inline int ring_depth(int bm, int cg) {
  const int fixed = smem_map(bm, cg, 0).total;
  const int d = (227 * 1024 - fixed) / stage_bytes(bm, cg);
  return d < MAX_STAGES ? d : MAX_STAGES;
}

// How many clusters of 2 .. 8 CTAs that fill an SM each the GPU holds at once (a cluster stays within a GPC): of 148 SMs as the occupancy
// query counts them on a B200; other counts of SMs in proportion.
struct ClusterFit { int n[MAX_SPLIT + 1]; };
inline ClusterFit cluster_fit(int sm_count) {
  const int of_148[MAX_SPLIT + 1] = {0, 148, 74, 45, 33, 26, 22, 15, 15};
  ClusterFit f;
  for (int c = 0; c <= MAX_SPLIT; ++c) f.n[c] = of_148[c] * sm_count / 148;
  return f;
}

// Tile shape, and how the tiles are dealt out: the cheapest form by an estimate in clocks.  Its constants are fitted to 2067 timings, the forms of 110
// problems of 3 .. 8192 tokens; the forms it chooses take 1 % longer than the fastest on average, a tenth at worst.
inline Tiling choose_tiling(int M, int N, int K, int sm_count, const ClusterFit& fit) {
  const int nst = (K + BK - 1) / BK;
  Tiling best;
  memset(&best, 0, sizeof(best));
  double best_cost = 1e300;
  for (int cg = 1; cg <= (sm_count < 2 ? 1 : 2); ++cg) {
    const int P = sm_count / cg;
    const long long tn = (static_cast<long long>(N) + cg * BN - 1) / (cg * BN);
    const int step = 16 * cg;
    for (int bm = step; bm <= 256; bm += step) {
      const long long tm = (static_cast<long long>(M) + bm - 1) / bm;
      if (bm > step && tm == (static_cast<long long>(M) + bm - step - 1) / (bm - step)) continue;     // the same number of tiles fit a lower tile
      const long long tiles = tn * tm;
      Tiling t;
      t.cg = cg; t.bm = bm; t.tn = static_cast<int>(tn); t.tm = static_cast<int>(tm); t.n_tiles = static_cast<int>(tiles);
      t.group = 8;
      t.depth = ring_depth(bm, cg);
      // a stage: its MMAs (8192 products a clock and SM, and what power leaves of that), its copies from L2, the hand-over
      const auto stage = [&](int rows) {
        const double mma = 2.78 * rows, copies = stage_bytes(rows, cg) / 50.5, c = mma > copies ? mma : copies;
        return c > 411.0 ? c : 411.0;
      };
      // storing a tile: two groups of warps take its 32-column chunks in turn
      const auto store = [&](int rows) { return 2872.0 + (staged(bm) ? (N % 8 ? 2568.0 : 935.0) * ((rows + 63) / 64) : 0.0); };
      const auto tile_clocks = [&](int rows) { const double k = nst * stage(rows); return k > store(rows) ? k : store(rows); };
      const double memory = (static_cast<double>(N) * K + static_cast<double>(M) * K + 2.0 * M * N) / 11424.0;     // at this many bytes a clock from HBM and L2
      const double start = cg == 1 ? 3279.0 : 6125.0;
      const auto consider = [&](long long teams, long long full, int tail, int split, double work, double rest) {
        double used = 1.15 * static_cast<double>(teams) * cg / sm_count;
        if (used > 1.0) used = 1.0;
        const double cost = start + (work > memory / used ? work : memory / used) + rest;
        if (cost > best_cost) return;            // (of equal ones the higher tile)
        best_cost = cost;
        t.teams = static_cast<int>(teams); t.full = static_cast<int>(full); t.tail = tail; t.split = split;
        best = t;
      };
      const long long waves = tiles / P, rem = tiles % P;
      const long long whole = tiles < P ? tiles : P;
      consider(whole, tiles, 1, 1, static_cast<double>((tiles + whole - 1) / whole) * tile_clocks(bm), store(bm));
      if (rem == 0) continue;
      if (waves > 0) {
        for (int tail = 2; tail <= 8; tail *= 2) {
          const int piece = bm / tail;
          if (piece * tail != bm || piece % step != 0) continue;
          consider(P, tiles - rem, tail, 1, waves * tile_clocks(bm) + static_cast<double>((rem * tail + P - 1) / P) * tile_clocks(piece), store(piece));
        }
      } else if (cg == 1) {
        for (int c = 2; c <= MAX_SPLIT && c <= nst; ++c)
          if (tiles <= fit.n[c]) consider(tiles * c, tiles, 1, c, ((nst + c - 1) / c) * stage(bm), 4984.0 + 75.0 * bm);
      }
    }
  }
  // No more stages than a team has use for (and the cluster's exchange needs): a small call then leaves room on the SM for the next kernel's start.
  const long long stages = best.split > 1 ? (nst + best.split - 1) / best.split : (static_cast<long long>(best.n_tiles) + best.teams - 1) / best.teams * nst;
  const int exchange = best.split > 1 ? ((M < best.bm ? M : best.bm) + best.split - 1) / best.split * best.split * BN * 4 : 0;
  while (best.depth > 2 && best.depth > stages && (best.depth - 1) * stage_bytes(best.bm, best.cg) >= exchange) --best.depth;
  return best;
}

// Whether TMA can read the operand: rows on 16 bytes.
inline bool mappable(const void* p, long long ld) { return aligned(p, 16) && ld % 16 == 0; }

// A call: one product, or one for each piece of the weights that are copied first.
struct Plan {
  Tiling main, tail;         // of the pieces, and of a last one of fewer rows
  int piece, tail_rows;      // weight rows of a piece
  size_t x_copy, w_copy;
  // [shared counter region][x on 16 bytes][a piece of w on 16 bytes]
  size_t bytes() const { return x_copy + w_copy ? kWorkspaceCounterBytes + x_copy + w_copy : 0; }
};
inline Plan make_plan(int M, int N, int K, int sm_count, const ClusterFit& fit, bool x_mappable, bool w_mappable) {
  constexpr long long W_COPY = 48ll << 20;     // stays in L2 beside x and out
  const long long row = (static_cast<long long>(K) + 15) / 16 * 16;
  Plan q;
  memset(&q, 0, sizeof(q));
  q.piece = N;
  if (!w_mappable && N * row > W_COPY) {
    const long long pieces = (N * row + W_COPY - 1) / W_COPY;
    long long rows = ((N + pieces - 1) / pieces + 255) / 256 * 256;
    if (rows * row > W_COPY) rows = W_COPY / row / 256 * 256;        // (at least 256: rows are at most 128 KiB)
    if (rows < N) q.piece = static_cast<int>(rows);
  }
  q.tail_rows = N % q.piece;
  q.main = choose_tiling(M, q.piece, K, sm_count, fit);
  if (q.tail_rows) q.tail = choose_tiling(M, q.tail_rows, K, sm_count, fit);
  const auto up = [](long long n) { return static_cast<size_t>((n + 1023) / 1024 * 1024); };
  if (!x_mappable) q.x_copy = up(M * row);
  if (!w_mappable) q.w_copy = up(q.piece * row);
  return q;
}

inline Params make_params(const Tiling& t, int M, int N, int K) {
  Params p;
  memset(&p, 0, sizeof(p));
  p.M = M; p.N = N; p.K = K;
  p.bm = t.bm; p.tn = t.tn; p.tm = t.tm; p.n_tiles = t.n_tiles; p.group = t.group;
  p.nst = (K + BK - 1) / BK;
  p.teams = t.teams; p.full = t.full; p.tail = t.tail; p.split = t.split; p.depth = t.depth;
  p.piece_bm = t.bm / t.tail;
  p.by_tail = make_divisor(t.tail);
  p.by_group_tiles = make_divisor(t.group * t.tn);
  p.by_group = make_divisor(t.group);
  p.by_last_group = make_divisor(t.tm % t.group ? t.tm % t.group : t.group);
  p.tmem_cols = 32;                            // the epilogue reads 32 columns at a time
  while (p.tmem_cols < t.bm + (t.bm + 31) / 32 * 32) p.tmem_cols *= 2;
  return p;
}

// The shared memory of a launch.  A CTA waits without a limit for its columns of tensor memory, and the other CTAs of its cluster wait for it: two clusters
// of two streams that meet on two SMs in opposite order, each with columns that the other one wants, would wait for good.  So a cluster's CTAs take as much of an
// SM's 228 KB as of its 512 columns, and a little more: where the columns of several are too many, they do not fit on an SM together.
// (Asked for beyond the ring by pairs with K of 384 and less.)
constexpr int SMEM_PER_COLUMN = 440;           // 544 columns (the least that is too many): 233.75 KB
inline int launch_smem(const Params& p, int cg) {
  const int ring = smem_map(p.bm, cg, p.depth).total, columns = cg * p.split > 1 ? p.tmem_cols * SMEM_PER_COLUMN : 0;
  return ring > columns ? ring : columns;
}

template <int CG, typename OT>
int launch_t(const CUtensorMap* tm, const Params& p, cudaStream_t stream) {
  auto kern = int8_gemm_kernel<CG, OT>;
  static thread_local int configured_device = -1;
  int dev = 0;
  LCQ_CUDA_TRY(cudaGetDevice(&dev));
  if (configured_device != dev) {
    LCQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    configured_device = dev;
  }
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  gemm_tc::pdl_launch_config(cfg, attr, CG * p.teams, NTHREADS, launch_smem(p, CG), stream);
  const int cluster = CG == 2 ? 2 : p.split;
  if (cluster > 1) {
    cudaLaunchAttribute& a = attr[cfg.numAttrs++];
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = cluster;
    a.val.clusterDim.y = 1;
    a.val.clusterDim.z = 1;
  }
  LCQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tm[0], tm[1], tm[2], tm[3], p));
  return LCQ_OK;
}

struct Operands {
  const void* x; long long ldx;
  const float* x_scales;
  const void* w; long long ldw;
  const void* w_scales; int w_scale_dtype;
  void* out; long long ldo; int out_dtype;
};
// One product of operands that TMA can read.
inline int launch_tiling(const Tiling& t, const Operands& o, int M, int N, int K, cudaStream_t stream) {
  Params p = make_params(t, M, N, K);
  p.out = o.out;
  p.ldo = o.ldo;
  p.x_scales = o.x_scales;
  p.w_scales = o.w_scales;
  p.w_scale_dtype = o.w_scale_dtype;
  const int e = o.out_dtype == LCQ_F32 ? 4 : 2;
  p.vec = aligned(o.out, 16) && (o.ldo * e) % 16 == 0;
  CUtensorMap tm[4];         // x in whole tiles, x in pieces of a tile, weights, out
  memset(tm, 0, sizeof(tm));
  const uint64_t k64 = static_cast<uint64_t>(K), m64 = static_cast<uint64_t>(M), n64 = static_cast<uint64_t>(N);
  int rc = encode_tmap_2d(&tm[0], 0, o.x, k64, m64, static_cast<uint64_t>(o.ldx), BK, t.bm / t.cg, 3);
  if (rc != LCQ_OK) return rc;
  if (t.tail > 1 && (rc = encode_tmap_2d(&tm[1], 0, o.x, k64, m64, static_cast<uint64_t>(o.ldx), BK, t.bm / t.tail / t.cg, 3)) != LCQ_OK) return rc;
  if ((rc = encode_tmap_2d(&tm[2], 0, o.w, k64, n64, static_cast<uint64_t>(o.ldw), BK, BN, 3)) != LCQ_OK) return rc;
  if (p.vec && staged(t.bm) && (rc = encode_tmap_2d(&tm[3], e == 4 ? 3 : 1, o.out, n64, m64, static_cast<uint64_t>(o.ldo) * e, BN, OUT_BOX, 0)) != LCQ_OK)
    return rc;
  switch (o.out_dtype) {
    case LCQ_F32: return t.cg == 2 ? launch_t<2, float>(tm, p, stream) : launch_t<1, float>(tm, p, stream);
    case LCQ_F16: return t.cg == 2 ? launch_t<2, __half>(tm, p, stream) : launch_t<1, __half>(tm, p, stream);
    case LCQ_BF16: return t.cg == 2 ? launch_t<2, __nv_bfloat16>(tm, p, stream) : launch_t<1, __nv_bfloat16>(tm, p, stream);
    default: break;
  }
  set_error("int8 matmul: bad out_dtype %d", o.out_dtype);
  return LCQ_ERR_BAD_ARG;
}

struct Rows { const void* src; long long ld; void* dst; long long rows; };
// Copies up to 2^30 pieces of 16 bytes of each of two operands in a launch.
inline int launch_align(Rows a, Rows b, int K, int sm_count, cudaStream_t stream) {
  const int per_row = (K + 15) / 16;
  const long long most = (1ll << 30) / per_row;
  const auto take = [&](Rows& r) {
    const long long n = r.rows < most ? r.rows : most;
    const AlignJob job = {static_cast<const uint8_t*>(r.src), r.ld, static_cast<uint4*>(r.dst), static_cast<int>(n * per_row)};
    r.src = static_cast<const uint8_t*>(r.src) + n * r.ld;
    r.dst = static_cast<uint4*>(r.dst) + n * per_row;
    r.rows -= n;
    return job;
  };
  while (a.rows > 0 || b.rows > 0) {
    const AlignJob first = take(a), second = take(b);
    long long blocks = (static_cast<long long>(first.pieces) + second.pieces + 1023) / 1024;
    if (blocks > sm_count * 8ll) blocks = sm_count * 8ll;
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[1];
    gemm_tc::pdl_launch_config(cfg, attr, static_cast<int>(blocks), 256, 0, stream);
    LCQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, align_rows_kernel, first, second, K, per_row, make_divisor(per_row)));
  }
  return LCQ_OK;
}

inline int launch(Operands o, int M, int N, int K, void* workspace, size_t ws_bytes, int sm_count, const ClusterFit& fit, cudaStream_t stream) {
  const bool x_mappable = mappable(o.x, o.ldx), w_mappable = mappable(o.w, o.ldw);
  const Plan q = make_plan(M, N, K, sm_count, fit, x_mappable, w_mappable);
  const size_t need = q.bytes();
  if (need && (workspace == nullptr || ws_bytes < need || !aligned(workspace, 256))) {
    set_error("int8 matmul: workspace of %zu bytes (256-byte aligned) required, got %zu", need, ws_bytes);
    return LCQ_ERR_WORKSPACE;
  }
  uint8_t* scratch = need ? static_cast<uint8_t*>(workspace) + kWorkspaceCounterBytes : nullptr;
  const long long row = (static_cast<long long>(K) + 15) / 16 * 16;
  const Rows none = {nullptr, 0, nullptr, 0};
  const Rows x_rows = {o.x, o.ldx, scratch, M};
  if (!x_mappable) {
    o.x = scratch;
    o.ldx = row;
  }
  const uint8_t* w = static_cast<const uint8_t*>(o.w);
  const uint8_t* w_scales = static_cast<const uint8_t*>(o.w_scales);
  uint8_t* out = static_cast<uint8_t*>(o.out);
  const long long ldw = o.ldw;
  for (int n0 = 0; n0 < N; n0 += q.piece) {
    const int n = N - n0 < q.piece ? N - n0 : q.piece;
    const bool copy_x = !x_mappable && n0 == 0;
    if (copy_x || !w_mappable) {
      const Rows w_rows = {w + n0 * ldw, ldw, scratch + q.x_copy, n};
      const int rc = launch_align(copy_x ? x_rows : none, w_mappable ? none : w_rows, K, sm_count, stream);
      if (rc != LCQ_OK) return rc;
    }
    if (!w_mappable) {
      o.w = scratch + q.x_copy;
      o.ldw = row;
    }
    o.w_scales = w_scales + static_cast<size_t>(n0) * (o.w_scale_dtype == LCQ_F32 ? 4 : 2);
    o.out = out + static_cast<size_t>(n0) * (o.out_dtype == LCQ_F32 ? 4 : 2);
    const int rc = launch_tiling(n == q.piece ? q.main : q.tail, o, M, n, K, stream);
    if (rc != LCQ_OK) return rc;
    if (N - n0 <= q.piece) break;            // (n0 + piece may pass 2^31)
  }
  return LCQ_OK;
}

}  // namespace int8_gemm
}  // namespace lcq
