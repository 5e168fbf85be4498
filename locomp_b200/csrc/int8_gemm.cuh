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
// Split of the work: whole tiles in turn while they fill all teams; the rest is cut along K into equal shares, whose
// int32 partials meet through scratch (the last contributor adds them up; nobody waits for another CTA), or, where there
// are few tiles, a cluster of CTAs shares the K of each tile and adds up over distributed shared memory.
//
// The weights' first stages are fetched into L2 while the kernel before this one still runs.  L2 is where all SMs' stores
// meet, so this is right whoever writes the weights; everything is read after that kernel has completed.
//
// LOADER: operands whose rows do not start on 16 bytes (K % 16 != 0 in contiguous storage, or an odd offset) have no
// tensor map.  Eight warps fetch them in words, shift and store them where TMA would have put them.
//
// Every mbarrier wait is bounded; on expiry the kernel records a status code and unwinds.
#pragma once
#include "gemm_tc.cuh"

namespace lcq {
namespace int8_gemm {

using gemm_tc::Ring;
using gemm_tc::all_epilogue_warps;
using gemm_tc::arrive_leader;
using gemm_tc::cluster_barrier;
using gemm_tc::leader_addr;
using gemm_tc::load_acquire;
using gemm_tc::peer_addr;
using gemm_tc::store_remote;
using gemm_tc::tc_fence_after;
using gemm_tc::tc_fence_before;
using gemm_tc::tma_load_2d_pair;
using gemm_tc::tmem_alloc;
using gemm_tc::tmem_dealloc;
using gemm_tc::tmem_ld32;
using gemm_tc::tmem_wait_ld;
using gemm_tc::umma_commit;
using gemm_tc::wait_bar;
using gemm_tc::warp_wait;
using gemm_tc::BAR_EPI;

constexpr int BN = 128;                      // weight rows per CTA
constexpr int BK = 128;                      // k per stage: one swizzled row of 128 bytes, four MMAs
constexpr int W_STAGE = BN * BK;
constexpr int MAX_STAGES = 12;
constexpr int WARP_TMA = 4, WARP_MMA = 5, N_LOADERS = 8;     // warps 0 .. 3: epilogue
constexpr int MAX_K = 131071;
constexpr int MAX_SPLIT = 8;

__host__ __device__ constexpr int threads(bool loader) { return (6 + (loader ? N_LOADERS : 0)) * 32; }

struct Params {
  void* out;                 // [M, N]
  const float* x_scales;     // [M]
  const void* w_scales;      // [N]
  const uint8_t *x, *w;      // LOADER
  long long ldx, ldw;        // LOADER: bytes between rows
  int* partials;             // [2 * teams * CG][bm][BN]
  int* counters;             // [sk_tiles * CG], zero on entry, zero on exit
  int M, N, K, w_scale_dtype;
  int bm;                    // tokens per tile (MMA N): a multiple of 16 CG, at most 256
  int tn, tm, n_tiles;
  int group;                 // token tiles that are walked together
  int nst;                   // 128-k stages per tile
  int teams;                 // CTAs (CG = 1) or pairs (CG = 2) launched
  int sk_tiles;              // tiles 0 .. sk_tiles - 1 are cut along K, the others go whole to team (tile - sk_tiles) % teams
  int split;                 // > 1: a cluster of `split` CTAs per tile, each with its share of K
  int depth;                 // stages in the ring
  int tmem_cols;
};

__host__ __device__ inline unsigned share_begin(const Params& p, int team) {
  const unsigned long long units = static_cast<unsigned long long>(p.sk_tiles) * static_cast<unsigned>(p.nst);
  return static_cast<unsigned>(units * static_cast<unsigned>(team) / static_cast<unsigned>(p.teams));
}
__host__ __device__ inline int share_owner(const Params& p, unsigned unit) {
  const unsigned long long units = static_cast<unsigned long long>(p.sk_tiles) * static_cast<unsigned>(p.nst);
  return static_cast<int>((static_cast<unsigned long long>(unit + 1u) * static_cast<unsigned>(p.teams) - 1u) / units);
}

// The segments of one team: (tile, stages st0 .. st1 - 1).  Every role walks them in the same order.
struct Walk {
  unsigned u, u1;            // what is left of the team's share of the cut tiles
  int next_tile;
  int tile, st0, st1;
  int mt, nt;                // the tile's place
  __host__ __device__ Walk(const Params& p, int team) {
    if (p.split > 1) {
      const int t = team / p.split, r = team - t * p.split;
      u = static_cast<unsigned>(t * p.nst + p.nst * r / p.split);
      u1 = static_cast<unsigned>(t * p.nst + p.nst * (r + 1) / p.split);
      next_tile = p.n_tiles;
    } else {
      u = share_begin(p, team);
      u1 = share_begin(p, team + 1);
      next_tile = p.sk_tiles + team;
    }
  }
  __host__ __device__ bool next(const Params& p) {
    if (u < u1) {
      tile = static_cast<int>(u / static_cast<unsigned>(p.nst));
      st0 = static_cast<int>(u - static_cast<unsigned>(tile) * static_cast<unsigned>(p.nst));
      const unsigned left = u1 - u, in_tile = static_cast<unsigned>(p.nst - st0);
      const unsigned take = left < in_tile ? left : in_tile;
      st1 = st0 + static_cast<int>(take);
      u += take;
    } else {
      tile = next_tile;
      if (tile >= p.n_tiles) return false;
      next_tile += p.teams;
      st0 = 0;
      st1 = p.nst;
    }
    // `group` token tiles at a time against all channels, tokens first: what runs at the same time shares its operands in L2
    const int per_group = p.group * p.tn, g = tile / per_group, in = tile - g * per_group;
    const int rows = p.tm - g * p.group < p.group ? p.tm - g * p.group : p.group;
    nt = in / rows;
    mt = g * p.group + in - nt * rows;
    return true;
  }
};

enum { FLAG_ABORT, FLAG_SHARED, ISSUED_0, ISSUED_1, N_FLAGS };
struct Smem { int bars, tmem_slot, flags, total; };         // offsets from the 1024-byte aligned base; the ring comes first
__host__ __device__ inline int stage_bytes(int bm, int cg) { return W_STAGE + (bm / cg) * BK; }
__host__ __device__ inline Smem smem_map(int bm, int cg, int depth) {
  Smem s;
  s.bars = depth * stage_bytes(bm, cg);
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

// The bytes p .. p + 15 of which the first `valid` exist; the others read as zero.  Only words that hold a byte that exists are read.
__device__ __forceinline__ uint4 load_unaligned16(const uint8_t* p, int valid) {
  if (valid >= 16 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) return *reinterpret_cast<const uint4*>(p);
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 3);
  const uint32_t* a = reinterpret_cast<const uint32_t*>(p - off);
  uint32_t v[5];
#pragma unroll
  for (int j = 0; j < 5; ++j) v[j] = 4 * j < off + valid ? a[j] : 0u;
  uint32_t r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t word = __funnelshift_r(v[j], v[j + 1], off * 8);
    const int left = valid - 4 * j;
    r[j] = left >= 4 ? word : left <= 0 ? 0u : word & ((1u << (8 * left)) - 1u);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
// Up to `rows` rows of a stage (128 k from k0 on) into shared memory, in 128-byte swizzled rows, by 32 * N_LOADERS threads.
__device__ __forceinline__ void load_rows(uint8_t* dst, const uint8_t* src, long long ld, int row0, int rows, int rows_left, int k0, int K, int t) {
  constexpr int T = N_LOADERS * 32;
  for (int i0 = t; i0 < rows * 8; i0 += 4 * T) {
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * T, r = i >> 3, k = k0 + (i & 7) * 16;
      const bool there = i < rows * 8 && r < rows_left && k < K;
      v[j] = there ? load_unaligned16(src + (static_cast<long long>(row0) + r) * ld + k, K - k) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + j * T, r = i >> 3;
      if (i < rows * 8) *reinterpret_cast<uint4*>(dst + r * 128 + (((i & 7) ^ (r & 7)) << 4)) = v[j];
    }
  }
}

// After a wait ran out in the CTA or its partner: waits for what they still have under way (the MMAs, and the copies into the last
// stages, which nobody waits for any more).  A CTA of a pair may have loaded its part of a stage whose other part was
// never issued: the barrier is then given the missing part, or armed for the one that comes.  All threads; in a pair between two
// cluster barriers.
template <int CG, bool LOADER>
__device__ __noinline__ void drain(const Params& p, uint8_t* smem, uint32_t crank) {
  const Smem L = smem_map(p.bm, CG, p.depth);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.bars);
  uint64_t* drained = full + 2 * MAX_STAGES + 4;
  const volatile int* flags = reinterpret_cast<const volatile int*>(smem + L.flags);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (warp == WARP_MMA) {
    if (crank == 0) umma_commit<CG>(drained);
    __syncwarp();
    mbar_wait_landed(drained, 0);
  } else if (!LOADER && warp == WARP_TMA && lane == 0 && crank == 0) {
    const int mine = flags[ISSUED_0], other = CG == 2 ? flags[ISSUED_1] : mine, n = mine > other ? mine : other;
    const int bytes = stage_bytes(p.bm, CG);
    for (int i = n > p.depth ? n - p.depth : 0; i < n; ++i) {
      uint64_t* bar = full + i % p.depth;
      if (i >= mine) mbar_expect_tx(bar, bytes);
      else if (i >= other) asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
      mbar_wait_landed(bar, (i / p.depth) & 1);
    }
  }
  __syncthreads();
}

// 32 columns (tokens) of a tile from column c0 on: this lane's channel of each.
template <typename OT>
__device__ __forceinline__ void store_columns(const uint32_t (&v)[32], OT* out, long long N, bool there, int c0, int rows, const float* x_scales, float ws, int lane) {
  const float xs = c0 + lane < rows ? x_scales[c0 + lane] : 0.0f;
  OT* o = out + static_cast<long long>(c0) * N;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float s = __shfl_sync(0xffffffffu, xs, i);
    if (there && c0 + i < rows) *o = from_f32<OT>(static_cast<float>(static_cast<int>(v[i])) * s * ws);
    o += N;
  }
}

template <int CG, typename OT, bool LOADER>
__global__ void __launch_bounds__(threads(LOADER), 1)
int8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ Params p) {
  static_assert(!(LOADER && CG == 2), "the loader form runs on single SMs");
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
    for (int i = 0; i < MAX_STAGES; ++i) { mbar_init(&full[i], LOADER ? N_LOADERS : 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&full_d[i], 1); mbar_init(&empty_d[i], 4 * CG); }
    mbar_init(drained, 1);
    *flag_abort = 0;
    fence_barrier_init();
    griddep_launch_dependents();
  }
  if (!LOADER && warp == WARP_TMA && lane == 0) {
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
  const uint32_t tmem_base = *tmem_slot;

#define LCQ_GIVE_UP(code)                                                                              \
  do {                                                                                                 \
    *flag_abort = 1;                                                                                   \
    if (CG == 2) store_remote(peer_addr(smem_u32(smem + L.flags + 4 * FLAG_ABORT), crank ^ 1u), 1);    \
    atomicExch(&g_device_status, (code));                                                              \
  } while (0)

  if (warp == WARP_TMA) {
    // ------------------------------------------------------------ this CTA's weight rows and tokens of each stage
    if (!LOADER && lane == 0) {
      griddep_wait();
      const int rows = p.bm / CG;
      Ring r = {0, 0};
      bool ok = true;
      int issued = 0;
      for (Walk w(p, team); ok && w.next(p);) {
        const int n0 = w.nt * (CG * BN) + static_cast<int>(crank) * BN, m0 = w.mt * p.bm + static_cast<int>(crank) * rows;
        for (int st = w.st0; st < w.st1; ++st, r.step(p.depth)) {
          if (!wait_bar(flag_abort, &empty[r.i], r.phase ^ 1u)) { LCQ_GIVE_UP(60); ok = false; break; }
          uint8_t* dst = smem + r.i * stage;
          if (crank == 0) mbar_expect_tx(&full[r.i], CG * stage);
          if (CG == 2) {
            const uint32_t bar = leader_addr<CG>(full + r.i);
            tma_load_2d_pair(dst, &tmap_w, bar, st * BK, n0);
            tma_load_2d_pair(dst + W_STAGE, &tmap_x, bar, st * BK, m0);
          } else {
            tma_load_2d(dst, &tmap_w, full + r.i, st * BK, n0);
            tma_load_2d(dst + W_STAGE, &tmap_x, full + r.i, st * BK, m0);
          }
          ++issued;
        }
      }
      if (CG == 2) store_remote(peer_addr(smem_u32(smem + L.flags + 4 * (ISSUED_0 + crank)), 0), issued);
      else flag_abort[ISSUED_0] = issued;
    }
  } else if (warp == WARP_MMA) {
    // ------------------------------------------------------------ MMA issuer: one warp for the team
    if (crank == 0) {
      const uint32_t desc0 = gemm_tc::make_b_desc(smem_u32(smem));             // descriptors count 16-byte units
      const uint32_t idesc = make_idesc(p.bm, CG);
      Ring r = {0, 0}, rd = {0, 0};
      bool ok = true;
      for (Walk w(p, team); ok && w.next(p); rd.step(2)) {
        if (!warp_wait(flag_abort, &empty_d[rd.i], rd.phase ^ 1u)) { if (lane == 0) LCQ_GIVE_UP(61); ok = false; break; }
        tc_fence_after();
        const uint32_t d_t = tmem_base + rd.i * p.bm;
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
  } else if (warp < WARP_TMA) {
    // ------------------------------------------------------------ epilogue warps: TMEM -> global
    griddep_wait();                            // out and the scratch may still be in the preceding kernel's use
    const int r = warp * 32 + lane;
    const uint32_t lane_taddr = tmem_base + (static_cast<uint32_t>(warp * 32) << 16);
    const uint32_t empty_d0 = leader_addr<CG>(empty_d);
    volatile int* shared_int = flag_abort + FLAG_SHARED;
    const long long part_elems = static_cast<long long>(p.bm) * BN;
    Ring rd = {0, 0};
    for (Walk w(p, team); w.next(p); rd.step(2)) {
      const int n = w.nt * (CG * BN) + static_cast<int>(crank) * BN + r, m0 = w.mt * p.bm;
      const bool there = n < p.N;
      const uint32_t d_t = lane_taddr + rd.i * p.bm;
      const int rows = p.M - m0 < p.bm ? p.M - m0 : p.bm;
      const float ws = there ? load_scale(p.w_scales, n, p.w_scale_dtype) : 0.0f;
      const float* xs = p.x_scales + m0;
      OT* out = static_cast<OT*>(p.out) + static_cast<long long>(m0) * p.N + n;
      if (!all_epilogue_warps(wait_bar(flag_abort, &full_d[rd.i], rd.phase))) { if (lane == 0) LCQ_GIVE_UP(63); break; }
      tc_fence_after();
      if (CG == 1 && p.split > 1) break;       // the cluster adds up its shares below
      // who else contributes to this tile: teams p0 .. p1
      int p0 = team, p1 = team, slot1 = 0;
      if (w.tile < p.sk_tiles) {
        const unsigned t0 = static_cast<unsigned>(w.tile) * static_cast<unsigned>(p.nst);
        p0 = share_owner(p, t0);
        p1 = share_owner(p, t0 + static_cast<unsigned>(p.nst) - 1u);
        slot1 = share_begin(p, p0) < t0;       // p0 came from the tile before (slot 0); the others' shares begin here
      }
      const auto part = [&](int q) {
        return p.partials + (static_cast<long long>(2 * q + (q == p0 ? slot1 : 0)) * CG + crank) * part_elems + r;
      };
      bool finish = p1 == p0;
      int* counter = p.counters + w.tile * CG + crank;
      if (!finish) {
        // published already by all the others?  Then this CTA finishes the tile without publishing.
        if (threadIdx.x == 0) *shared_int = load_acquire(counter);
        named_bar_sync(BAR_EPI, 128);
        finish = *shared_int == p1 - p0;
        named_bar_sync(BAR_EPI, 128);
        if (!finish) {
          int* mine = part(team);
          for (int c0 = 0; c0 < rows; c0 += 32) {
            uint32_t v[32];
            tmem_ld32(d_t + c0, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c0 + i < rows) __stcg(mine + (c0 + i) * BN, static_cast<int>(v[i]));
          }
          __threadfence();
          named_bar_sync(BAR_EPI, 128);
          if (threadIdx.x == 0) *shared_int = atomicAdd(counter, 1);
          named_bar_sync(BAR_EPI, 128);
          finish = *shared_int == p1 - p0;
          named_bar_sync(BAR_EPI, 128);
        }
        __threadfence();
      }
      if (finish) {
        for (int c0 = 0; c0 < rows; c0 += 32) {
          uint32_t v[32];
          tmem_ld32(d_t + c0, v);
          tmem_wait_ld();
          for (int q = p0; q <= p1; ++q) {
            if (q == team) continue;
            const int* src = part(q) + c0 * BN;
            int u[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] = c0 + i < rows ? __ldcg(src + i * BN) : 0;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] += static_cast<uint32_t>(u[i]);
          }
          store_columns<OT>(v, out, p.N, there, c0, rows, xs, ws, lane);
        }
        if (p1 != p0 && threadIdx.x == 0) *counter = 0;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_leader<CG>(empty_d0 + rd.i * 8);
    }
  } else if (LOADER) {
    // ------------------------------------------------------------ loader warps: words -> swizzled rows
    griddep_wait();
    const int t = threadIdx.x - (WARP_MMA + 1) * 32;
    Ring r = {0, 0};
    bool ok = true;
    for (Walk w(p, team); ok && w.next(p);) {
      const int n0 = w.nt * BN, m0 = w.mt * p.bm;
      for (int st = w.st0; st < w.st1; ++st, r.step(p.depth)) {
        if (!warp_wait(flag_abort, &empty[r.i], r.phase ^ 1u)) { if (lane == 0) LCQ_GIVE_UP(64); ok = false; break; }
        uint8_t* dst = smem + r.i * stage;
        load_rows(dst, p.w, p.ldw, n0, BN, p.N - n0, st * BK, p.K, t);
        load_rows(dst + W_STAGE, p.x, p.ldx, m0, p.bm, p.M - m0, st * BK, p.K, t);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");           // the MMAs read through the async proxy
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[r.i]);
      }
    }
  }
#undef LCQ_GIVE_UP

  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_barrier();    // neither CTA leaves while the other may still arrive on its barriers or the pair's MMAs read its memory
  if (*flag_abort) {
    drain<CG, LOADER>(p, smem, crank);
    if (CG == 2) cluster_barrier();
  }
  if (CG == 1 && p.split > 1) {
    // One tile per cluster, its K shared out: CTA d settles columns d * cw .. of the tile.  Every CTA sends each of the others its
    // part of their columns (into the ring, which nobody uses any more).
    Walk w(p, team);
    w.next(p);
    const int me = team % p.split, m0 = w.mt * p.bm;
    const int rows = p.M - m0 < p.bm ? p.M - m0 : p.bm;
    const int cw = (rows + p.split - 1) / p.split;
    const int r = warp * 32 + lane;
    cluster_barrier();
    if (warp < WARP_TMA) {
      tc_fence_after();
      const uint32_t mine = smem_u32(smem) + (me * cw * BN + r) * 4;
      for (int c0 = 0; c0 < rows; c0 += 32) {
        uint32_t v[32];
        tmem_ld32(tmem_base + (static_cast<uint32_t>(warp * 32) << 16) + c0, v);
        tmem_wait_ld();
        int d = c0 / cw, j = c0 - d * cw;
        uint32_t dst = peer_addr(mine + j * (BN * 4), d);
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if (c0 + i < rows) store_remote(dst, static_cast<int>(v[i]));
          dst += BN * 4;
          if (++j == cw && d + 1 < p.split) { j = 0; ++d; dst = peer_addr(mine, d); }
        }
      }
      tc_fence_before();
    }
    cluster_barrier();
    const int n = w.nt * BN + r;
    if (warp < WARP_TMA && n < p.N && *flag_abort == 0) {
      const int* got = reinterpret_cast<const int*>(smem) + r;
      const float ws = load_scale(p.w_scales, n, p.w_scale_dtype);
      OT* out = static_cast<OT*>(p.out) + static_cast<long long>(m0 + me * cw) * p.N + n;
      for (int j = 0; j < cw && me * cw + j < rows; ++j) {
        int sum = 0;
        for (int q = 0; q < p.split; ++q) sum += got[(q * cw + j) * BN];
        out[static_cast<long long>(j) * p.N] = from_f32<OT>(static_cast<float>(sum) * p.x_scales[m0 + me * cw + j] * ws);
      }
    }
  }
  if (warp == WARP_MMA) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc<CG>(tmem_base, p.tmem_cols);
  }
}

// ---------------------------------------------------------------------------- host side
struct Tiling { int cg, bm, tn, tm, n_tiles, group, teams, sk_tiles, split, depth; };

inline int ring_depth(int bm, int cg) {
  const int fixed = smem_map(bm, cg, 0).total + 1024;
  const int d = (227 * 1024 - fixed) / stage_bytes(bm, cg);
  return d < MAX_STAGES ? d : MAX_STAGES;
}

// Clocks of a 128-k stage of a tile: the MMAs (8192 products a clock and SM), the reads of the weight rows from shared memory, and the
// copies into the ring.
inline double stage_clocks(int cg, int bm) {
  const double mma = 2.0 * bm, copies = stage_bytes(bm, cg) / 48.0;
  const double c = mma > copies ? mma : copies;
  return c > 140.0 ? c : 140.0;
}

inline Tiling choose_tiling(int M, int N, int K, int sm_count, bool loader) {
  const int nst = (K + BK - 1) / BK;
  Tiling best;
  memset(&best, 0, sizeof(best));
  double best_cost = 1e300;
  for (int cg = 1; cg <= (loader || sm_count < 2 ? 1 : 2); ++cg) {
    const int P = sm_count / cg;
    const long long tn = (static_cast<long long>(N) + cg * BN - 1) / (cg * BN);
    const int step = 16 * cg;
    for (int bm = step; bm <= 256; bm += step) {
      const long long tm = (static_cast<long long>(M) + bm - 1) / bm;
      if (bm > step && tm == (static_cast<long long>(M) + bm - step - 1) / (bm - step)) continue;     // the same number of tiles fit a lower tile
      const long long tiles = tn * tm;
      Tiling t;
      t.cg = cg; t.bm = bm; t.tn = static_cast<int>(tn); t.tm = static_cast<int>(tm); t.n_tiles = static_cast<int>(tiles);
      t.group = bm >= 128 ? 8 : 16;
      t.depth = ring_depth(bm, cg);
      const double per = stage_clocks(cg, bm);
      const auto consider = [&](long long teams, long long sk, int split, double cost) {
        if (cost >= best_cost) return;
        best_cost = cost;
        t.teams = static_cast<int>(teams); t.sk_tiles = static_cast<int>(sk); t.split = split;
        best = t;
      };
      const long long waves = tiles / P, rem = tiles % P;
      const double start = cg == 1 ? 5000.0 : 5600.0;
      consider(tiles < P ? tiles : P, 0, 1, start + static_cast<double>(waves + (rem != 0)) * nst * per + 10.0 * bm);
      if (rem == 0) continue;
      // equal shares of K, with a wave of whole tiles added when the shares would be short
      const long long sk = rem * 3 >= P || waves == 0 ? rem : rem + P;
      const long long share = (sk * nst + P - 1) / P;
      if (nst > 1 && (waves == 0 || sk * nst >= P))       // (every team has a share)
        consider(P < sk * nst ? P : sk * nst, sk, 1, start + static_cast<double>((tiles - sk) / P) * nst * per + share * per + 3000.0 + 40.0 * bm);
      if (cg == 1 && waves == 0) {
        for (int c = 2; c <= MAX_SPLIT && c <= nst; ++c) {
          if (tiles > static_cast<long long>(sm_count / 18) * (16 / c)) continue;
          consider(tiles * c, 0, c, start + ((nst + c - 1) / c) * per + 1500.0 + 12.0 * bm);
        }
      }
    }
  }
  return best;
}

inline size_t partial_bytes(const Tiling& t) {
  return t.sk_tiles ? static_cast<size_t>(t.teams) * 2 * t.cg * t.bm * BN * sizeof(int) : 0;
}
// [shared counter region][int32 partials of the tiles cut along K]
inline size_t workspace_bytes(const Tiling& t) { return t.sk_tiles ? kWorkspaceCounterBytes + partial_bytes(t) : 0; }

// Whether TMA can read the operand: rows on 16 bytes.
inline bool mappable(const void* p, long long ld) { return aligned(p, 16) && ld % 16 == 0; }

inline Params make_params(const Tiling& t, int M, int N, int K) {
  Params p;
  memset(&p, 0, sizeof(p));
  p.M = M; p.N = N; p.K = K;
  p.bm = t.bm; p.tn = t.tn; p.tm = t.tm; p.n_tiles = t.n_tiles; p.group = t.group;
  p.nst = (K + BK - 1) / BK;
  p.teams = t.teams; p.sk_tiles = t.sk_tiles; p.split = t.split; p.depth = t.depth;
  p.tmem_cols = 32;                            // the epilogue reads 32 columns at a time
  while (p.tmem_cols < t.bm + (t.bm + 31) / 32 * 32) p.tmem_cols *= 2;
  return p;
}

template <int CG, typename OT, bool LOADER>
int launch_t(const CUtensorMap* tm, const Params& p, cudaStream_t stream) {
  auto kern = int8_gemm_kernel<CG, OT, LOADER>;
  static thread_local int configured_device = -1;
  int dev = 0;
  LCQ_CUDA_TRY(cudaGetDevice(&dev));
  if (configured_device != dev) {
    LCQ_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    configured_device = dev;
  }
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr[2];
  gemm_tc::pdl_launch_config(cfg, attr, CG * p.teams, threads(LOADER), smem_map(p.bm, CG, p.depth).total, stream);
  const int cluster = CG == 2 ? 2 : p.split;
  if (cluster > 1) {
    cudaLaunchAttribute& a = attr[cfg.numAttrs++];
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = cluster;
    a.val.clusterDim.y = 1;
    a.val.clusterDim.z = 1;
  }
  LCQ_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, tm[0], tm[1], p));
  return LCQ_OK;
}
template <typename OT>
int launch_by_form(int cg, bool loader, const CUtensorMap* tm, const Params& p, cudaStream_t stream) {
  if (loader) return launch_t<1, OT, true>(tm, p, stream);
  return cg == 2 ? launch_t<2, OT, false>(tm, p, stream) : launch_t<1, OT, false>(tm, p, stream);
}

inline int launch_tiling(const Tiling& t, const void* x, long long ldx, const void* x_scales, const void* w, long long ldw, const void* w_scales,
                         void* out, int M, int N, int K, int w_scale_dtype, int out_dtype, bool loader, void* workspace, size_t ws_bytes,
                         cudaStream_t stream) {
  const size_t need = workspace_bytes(t);
  if (need && (workspace == nullptr || ws_bytes < need || !aligned(workspace, 256))) {
    set_error("int8 matmul: workspace of %zu bytes (256-byte aligned) required, got %zu", need, ws_bytes);
    return LCQ_ERR_WORKSPACE;
  }
  Params p = make_params(t, M, N, K);
  p.out = out;
  p.x_scales = static_cast<const float*>(x_scales);
  p.w_scales = w_scales;
  p.w_scale_dtype = w_scale_dtype;
  p.x = static_cast<const uint8_t*>(x); p.ldx = ldx;
  p.w = static_cast<const uint8_t*>(w); p.ldw = ldw;
  p.counters = static_cast<int*>(workspace);
  p.partials = need ? reinterpret_cast<int*>(static_cast<uint8_t*>(workspace) + kWorkspaceCounterBytes) : nullptr;
  CUtensorMap tm[2];
  memset(tm, 0, sizeof(tm));
  if (!loader) {
    const uint64_t k64 = static_cast<uint64_t>(K);
    // (a single row has no row stride: any multiple of 16 that covers it will do)
    int rc = encode_tmap_2d(&tm[0], 0, x, k64, static_cast<uint64_t>(M), static_cast<uint64_t>(ldx), BK, t.bm / t.cg, 3);
    if (rc != LCQ_OK) return rc;
    if ((rc = encode_tmap_2d(&tm[1], 0, w, k64, static_cast<uint64_t>(N), static_cast<uint64_t>(ldw), BK, BN, 3)) != LCQ_OK) return rc;
  }
  switch (out_dtype) {
    case LCQ_F32: return launch_by_form<float>(t.cg, loader, tm, p, stream);
    case LCQ_F16: return launch_by_form<__half>(t.cg, loader, tm, p, stream);
    case LCQ_BF16: return launch_by_form<__nv_bfloat16>(t.cg, loader, tm, p, stream);
    default: break;
  }
  set_error("int8 matmul: bad out_dtype %d", out_dtype);
  return LCQ_ERR_BAD_ARG;
}

}  // namespace int8_gemm
}  // namespace lcq
