// Block attention of a batch whose requests share a prefix, on the 5th-generation tensor cores: every query of request b sees the
// shared prefix's pages and then the request's own, all of their keys (no mask but the lengths).
//
//   o = sum_j exp(q.k_j scale) v_j / sum_j exp(q.k_j scale),   lse = log sum_j exp(q.k_j scale)      over prefix ++ own keys
//
// The prefix is read once for all requests: their rows lie behind one another (row = token * group + head in group, tokens of all
// requests), so that against the prefix the batch is one dense product of many rows, bound by the tensor cores and the
// exponentials, while the requests' own keys are bound by memory.  Sums over parts of the keys are joined by their maxima (attn_shared_merge).
//
// A unit is one or two tiles of 128 rows of a key head (two walk the same key tiles, one's softmax under the other's products)
// against the prefix, or against one request's own keys.  All units' key tiles form one list in units of time; every CTA takes
// an equal run of it, so that no SM is left behind whatever the lengths, which the device alone knows.  The part that starts
// a unit leaves its sums (max, sum, O: fp32) at the rows' place, a part that goes on with one at its CTA's place (a CTA has one
// such part at most: its first); info[unit] says how many CTAs follow.
//
// Roles: a warp that works out the CTA's parts and hands them on through shared memory, a TMA warp (query tiles, rings of K and V
// tiles), an MMA warp, two groups of four softmax warps, a row per thread.  Units of two tiles take
// both groups; units of one take them in turn, each with the query tile, the output columns and the barriers of its group, so that
// one's start lies under the other's end.
// Tensor memory: S_0 (P_0) | S_1 (P_1) | O_0 | O_1, 128 columns each.  Of two tiles each has its score columns, of one it takes both in
// turn, the next scores ahead of P V.  P goes back into the columns its scores came from, in two halves, of which the first is
// multiplied while the second is made.  The products of one thread run in the order of issue, so scores may follow a P V into
// the same columns without a wait.
//
// What bounds it.  Two tiles: the chain scores -> maximum and weights (2050 cycles) -> products and next scores (1450), 3500 cycles a round for
// 2100 of products, and the power limit: 64 blocks of 32 tokens, 16 query and 8 key heads, behind 16384 keys and 1024 to 2048 own ones 322 us
// alone (930 TFLOP/s), 387 in a loop at 1.5 GHz.  One tile: memory, 64 x 16384 own keys at 5.9 TB/s.  A small batch: latency, 17 us for four
// blocks behind 1056 keys, of which the joining kernel 5.  No gain from a polynomial for some of the exponentials, nor from other
// splits of P.
// Where it pays: the block attention over tables that all begin with the prefix's pages (attention_tc.cu) reads the prefix once per request, but starts
// and joins faster.  16 query and 8 key heads, 300 own keys, us (this : that) for single tokens 4 x 2048 prefix keys 15 : 12, 4 x 4096 16 : 16,
// 8 x 2048 15 : 17, 32 x 512 20 : 24, 32 x 8192 28 : 140; blocks of 32 tokens 4 x 1024 16 : 12, 8 x 1024 16 : 17, 4 x 8192 24 : 26, 16 x 2048 26 : 25,
// 16 x 4096 34 : 40, 32 x 512 31 : 24, 32 x 2048 43 : 46, 32 x 8192 88 : 150.
#include "mdb_common.cuh"

namespace mdb {

// Times: a key tile of one query tile, of two, start and end of a unit; the least share of a CTA.  (5 : 8 : 6 for 6 : 8 : 10, 32 blocks
// behind 8192 keys: 92 for 95 us; 64 tokens behind 16384: 100 for 103.)
constexpr uint32_t kShOneStep = 5, kShTwoStep = 8, kShUnit = 6, kShMinShare = 16;

struct ShPlan {
  static constexpr int kKStages = 3, kVStages = 2;
  static constexpr int kQBytes = 2 * 128 * 128;            // a tile: two channel halves of [128 rows][128 B]
  static constexpr int kThreads = 384;                     // eight softmax warps, TMA, MMA, parts; one idle
  static constexpr int kParts = 4;                         // handed on ahead
  static constexpr int kSoftmaxRegs = 224, kOtherRegs = 56;       // (216 and 72: 331 for 321 us, 64 blocks of 32 behind 16384 keys)
  static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * 168, "registers after the split");
  static constexpr int kOffK = 2 * kQBytes;
  static constexpr int kOffV = kOffK + kKStages * kAtTileBytes;
  static constexpr int kOffBars = kOffV + kVStages * kAtTileBytes;
  static constexpr int kOffParts = kOffBars + 384, kPartBytes = 48;
  static constexpr int kSmemBytes = 1024 + kOffParts + kParts * kPartBytes;
};
static_assert(ShPlan::kSmemBytes <= 227 * 1024, "shared memory of the shared-prefix attention");

struct ShArgs {
  bf16* out;
  float* lse;                    // [tokens][hq], may be NULL
  const int32_t* prefix_len;
  const int32_t* prefix_table;
  const int32_t* ctx_lens;
  const int32_t* block_table;
  int prefix_pages, table_stride, table_pages, num_pages;
  int bs, block, hq, hkv, group;
  int tokens, rows;              // bs * block; rows of a key head: tokens * group
  int box_p, per_p, units_p;     // against the prefix: tokens of a query tile, tiles per unit, units per key head
  int box_o, per_o, units_o;     // against a request's own keys
  float scale_log2;
  // sums of parts lie [channels / 4][rows] of float4: neighbouring rows, neighbouring threads
  float4* main_o;                // [2: prefix, own][hkv][32][rows]
  float2* main_ml;               // [2][hkv][rows]: maximum in log2 units, sum
  float4* cont_o;                // [CTA][32][256]
  float2* cont_ml;               // [CTA][256]
  int2* info;                    // [hkv * units_p + bs * hkv * units_o]: CTA of the first part, how many follow
  int ctas;                      // of the launch that leaves the sums: places in cont_o and cont_ml
};

// of a group x: Q, O and P V barriers; S and P barriers by group and score columns
enum {
  kShBarQFull = 0, kShBarQEmpty = 2, kShBarKFull = 4, kShBarKEmpty = 7, kShBarVFull = 10, kShBarVEmpty = 12, kShBarSFull = 14 /* 2 x + buf */,
  kShBarPDone = 18, kShBarOFull = 20, kShBarOEmpty = 22, kShBarPFull = 24 /* 2 (2 x + buf) + half */, kShBarPartFull = 32,
  kShBarPartEmpty = 36, kShBarEnd = 40 /* of all products */, kShBarCount = 41
};

__device__ __forceinline__ int sh_prefix(const ShArgs& a) {
  return a.prefix_len == nullptr ? 0 : static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(*a.prefix_len), static_cast<int64_t>(a.prefix_pages) * kPage)));
}
__device__ __forceinline__ int sh_len(const ShArgs& a, int b) {
  return static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(a.ctx_lens[b]), static_cast<int64_t>(a.table_pages) * kPage)));
}
__device__ __forceinline__ uint32_t sh_steps(int len) { return (static_cast<uint32_t>(len) + kAtKeys - 1) / kAtKeys; }
__device__ __forceinline__ uint32_t sh_cost(uint32_t steps, int per) { return steps == 0 ? 0u : steps * (per == 2 ? kShTwoStep : kShOneStep) + kShUnit; }
// Key tiles of a unit in front of the time x since its start.
__device__ __forceinline__ uint32_t sh_cut(uint32_t x, uint32_t steps, int per) {
  if (x <= kShUnit) return 0u;
  x -= kShUnit;
  return min(steps, per == 2 ? (x + kShTwoStep / 2) / kShTwoStep : (x + kShOneStep / 2) / kShOneStep);
}

// A part of a unit.
struct __align__(16) ShPart {
  int req;                 // -1: the prefix
  int kvh, tok0;           // first token of the first tile (of all requests' tokens)
  int two;                 // there is a second tile
  int slot;                // group of a unit of one tile
  int tok_end, box;        // the rows end here; tokens of a tile
  int len, k0, k1;         // keys of the unit; key tiles of the part (k1 0: there are no more parts)
  int unit, followers;     // place in info; CTAs behind this one that have a part of the unit
};
static_assert(sizeof(ShPart) == ShPlan::kPartBytes, "a part's size");

// A CTA's run of the list.
struct ShWalk {
  uint32_t x0, x1, at;           // run, start of the unit at the cursor
  uint32_t per, rest, share;     // length of the list = per * share + rest, over so many CTAs
  int plen, len;                 // of the prefix, of the request at the cursor
  int b, kvh, u;                 // cursor: request (-1: prefix), key head, unit
  int turn;                      // group of the next unit of one tile
  __device__ __forceinline__ uint32_t start_of(uint32_t c) const { return per * c + min(c, rest); }
  // by a whole warp
  __device__ __forceinline__ void start(const ShArgs& a) {
    const int lane = threadIdx.x & 31;
    const uint32_t mine = lane < a.bs ? sh_cost(sh_steps(sh_len(a, lane)), a.per_o) : 0u;
    plen = sh_prefix(a);
    uint32_t own = mine;
    for (int i = lane + 32; i < a.bs; i += 32) own += sh_cost(sh_steps(sh_len(a, i)), a.per_o);
    own = __reduce_add_sync(0xffffffffu, own);
    const uint32_t cost_p = sh_cost(sh_steps(plen), a.per_p), per_req = static_cast<uint32_t>(a.hkv * a.units_o);
    const uint32_t all_p = cost_p * static_cast<uint32_t>(a.hkv * a.units_p), total = all_p + own * per_req;
    share = min(gridDim.x, max(1u, total / kShMinShare));
    per = total / share;
    rest = total - per * share;
    x0 = x1 = at = 0;
    b = -1; kvh = 0; u = 0; len = 0; turn = 0;
    if (blockIdx.x >= share) return;
    x0 = start_of(blockIdx.x);
    x1 = start_of(blockIdx.x + 1);
    if (x0 < all_p) {
      const uint32_t i = x0 / cost_p;
      at = i * cost_p;
      kvh = static_cast<int>(i) / a.units_p;
      u = static_cast<int>(i) - kvh * a.units_p;
      return;
    }
    at = all_p;
    for (int b0 = 0; b0 < a.bs; b0 += 32) {
      const uint32_t c = b0 == 0 ? mine : b0 + lane < a.bs ? sh_cost(sh_steps(sh_len(a, b0 + lane)), a.per_o) : 0u;
      uint32_t upto = c * per_req;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, x0 < at + upto);
      if (hit) {
        const int l = __ffs(hit) - 1;
        b = b0 + l;
        const uint32_t each = __shfl_sync(0xffffffffu, c, l);
        at += __shfl_sync(0xffffffffu, upto, l) - each * per_req;
        const uint32_t i = (x0 - at) / each;
        at += i * each;
        kvh = static_cast<int>(i) / a.units_o;
        u = static_cast<int>(i) - kvh * a.units_o;
        len = sh_len(a, b);
        return;
      }
      at += __shfl_sync(0xffffffffu, upto, 31);
    }
    x1 = x0;                     // (an empty list)
  }
  __device__ __forceinline__ bool next(const ShArgs& a, ShPart& p) {
    while (at < x1) {
      const bool prefix = b < 0;
      const int units = prefix ? a.units_p : a.units_o, tiles = prefix ? a.per_p : a.per_o, n = prefix ? plen : len;
      const uint32_t steps = sh_steps(n);
      if (steps == 0 || kvh == a.hkv) {                    // behind the units of the prefix or of a request
        if (++b >= a.bs) return false;
        kvh = 0; u = 0;
        len = sh_len(a, b);
        continue;
      }
      const uint32_t cost = sh_cost(steps, tiles);
      p.k0 = x0 <= at ? 0 : static_cast<int>(sh_cut(x0 - at, steps, tiles));
      p.k1 = static_cast<int>(x1 >= at + cost ? steps : sh_cut(x1 - at, steps, tiles));
      p.req = b;
      p.kvh = kvh;
      p.unit = (prefix ? 0 : a.hkv * (a.units_p + b * a.units_o)) + kvh * units + u;
      p.box = prefix ? a.box_p : a.box_o;
      p.tok0 = (prefix ? 0 : b * a.block) + u * tiles * p.box;
      p.tok_end = prefix ? a.tokens : (b + 1) * a.block;
      p.two = tiles == 2 && p.tok0 + p.box < p.tok_end;
      p.len = n;
      const uint32_t s = at;
      at += cost;
      if (++u == units) { u = 0; ++kvh; }
      if (p.k1 > p.k0) {
        p.slot = turn;
        if (!p.two) turn ^= 1;
        p.followers = 0;
        if (x1 < at)
          for (uint32_t c = blockIdx.x + 1; c < share; ++c, ++p.followers) {
            const uint32_t x = start_of(c);
            if (x >= at || sh_cut(x - s, steps, tiles) >= steps) break;
          }
        return true;
      }
    }
    return false;
  }
};

// Whether an entry of info names CTAs of the launch.  One that no CTA has written (a wait ran out) holds what the workspace held.
__host__ __device__ constexpr bool sh_info_there(int first, int followers, int ctas) {
  return first >= 0 && followers >= 0 && followers < ctas && first < ctas - followers;
}
static_assert(sh_info_there(0, 0, 1) && sh_info_there(0, 147, 148) && sh_info_there(147, 0, 148) && sh_info_there(100, 47, 148), "all CTAs of a launch");
static_assert(!sh_info_there(0, 1, 1) && !sh_info_there(148, 0, 148) && !sh_info_there(100, 48, 148) && !sh_info_there(1, 147, 148), "behind the last CTA");
static_assert(!sh_info_there(-1, -1, 148) && !sh_info_there(-1, 1, 148) && !sh_info_there(5, -1, 148) && !sh_info_there(0x5a5a5a5a, 0x5a5a5a5a, 148) &&
                  !sh_info_there(0x7fffffff, 0x7fffffff, 148) && !sh_info_there(0x7fffffff, 1, 148) && !sh_info_there(0, -0x7fffffff - 1, 148),
              "whatever lay there");

// The same number to one, eight or 32 columns of every lane.
__device__ __forceinline__ void tmem_fill1(uint32_t taddr, float v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "f"(v) : "memory");
}
__device__ __forceinline__ void tmem_fill8(uint32_t taddr, float v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %1, %1, %1, %1, %1, %1, %1};" ::"r"(taddr), "f"(v) : "memory");
}
__device__ __forceinline__ void tmem_fill32(uint32_t taddr, float v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, %1, "
      "%1, %1, %1, %1, %1, %1, %1, %1};" ::"r"(taddr), "f"(v)
      : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__global__ void __launch_bounds__(ShPlan::kThreads, 1)
attn_shared_kernel(const __grid_constant__ CUtensorMap map_qp, const __grid_constant__ CUtensorMap map_qo, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const ShArgs a) {
  using P = ShPlan;
  constexpr int kProducerWarp = 8, kMmaWarp = 9, kPartsWarp = 10;
  extern __shared__ __align__(1024) unsigned char sh_smem_raw[];
  const uint32_t raw = smem_u32(sh_smem_raw), base = (raw + 1023u) & ~1023u;
  unsigned char* gen_base = sh_smem_raw + (base - raw);
  const uint32_t bars = base + P::kOffBars;
  auto bar = [&](int slot) { return bars + 8u * static_cast<uint32_t>(slot); };
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(gen_base + P::kOffBars + 8 * kShBarCount);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_launch_dependents();
  if (warp == 0) {
    mbar_init(bar(lane), lane >= kShBarOEmpty ? 4 : 1);      // (the softmax warps' are the last ones of these)
    if (lane < kShBarCount - 32) mbar_init(bar(32 + lane), 32 + lane >= kShBarPartEmpty && 32 + lane < kShBarEnd ? 10 : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    const uint32_t slot = smem_u32(const_cast<uint32_t*>(&misc[0]));
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = misc[0];
  pdl_wait();
  ShPart* const parts = reinterpret_cast<ShPart*>(gen_base + P::kOffParts);
  ShPart w;
  AtRing part;
  // The next part (false: none, or `ok` is), by a warp or by its first thread.
  auto take = [&](bool& ok, uint32_t threads = 0xffffffffu) {
    ok = mbar_wait(bar(kShBarPartFull + part.stage), part.phase);
    ok = __all_sync(threads, ok);
    if (!ok) return false;
    const int4* from = reinterpret_cast<const int4*>(parts + part.stage);
    const int4 p0 = from[0], p1 = from[1];
    const int2 p2 = *reinterpret_cast<const int2*>(from + 2);
    w.req = p0.x; w.kvh = p0.y; w.tok0 = p0.z; w.two = p0.w;
    w.slot = p1.x; w.tok_end = p1.y; w.box = p1.z; w.len = p1.w;
    w.k0 = p2.x; w.k1 = p2.y;
    __syncwarp(threads);
    if (lane == 0) mbar_arrive(bar(kShBarPartEmpty + part.stage));
    part.advance(P::kParts);
    return w.k1 > 0;
  };

  if (warp >= kProducerWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P::kOtherRegs));
    if (warp == kProducerWarp) {
      // ------------------------------------------------------------------ producer
      if (lane == 0) {
        AtRing kr, vr;
        uint32_t q_phase = 0, pend_k = 0, pend_v = 0, pend_q = 0;     // stages with a copy in flight, and the parity it completes
        uint32_t par_k = 0, par_v = 0, par_q = 0;
        bool ok = true;
        auto load_tile = [&](const CUtensorMap* map, uint32_t tiles0, int full0, int empty0, int stages, AtRing& r, uint32_t& pend, uint32_t& par,
                             int kvh, int token_row) {
          if (!mbar_wait(bar(empty0 + r.stage), r.phase ^ 1)) return false;
          const uint32_t full = bar(full0 + r.stage), dst = tiles0 + r.stage * kAtTileBytes;
          mbar_arrive_expect_tx(full, 2 * kAtHalfBytes);
          tma_load_2d(dst, map, kvh * kHeadDim, token_row, full);
          tma_load_2d(dst + kAtHalfBytes, map, kvh * kHeadDim + 64, token_row, full);
          pend |= 1u << r.stage;
          par = (par & ~(1u << r.stage)) | (r.phase << r.stage);
          r.advance(stages);
          return true;
        };
        while (take(ok, 1u)) {
          const int32_t* table = w.req < 0 ? a.prefix_table : a.block_table + static_cast<int64_t>(w.req) * a.table_stride;
          int page = table[w.k0 * kAtKeys / kPage];
          const CUtensorMap* map_q = w.req < 0 ? &map_qp : &map_qo;
          for (int x = w.two ? 0 : w.slot; x <= (w.two ? 1 : w.slot); ++x) {
            if (!mbar_wait(bar(kShBarQEmpty + x), (q_phase >> x & 1) ^ 1)) { ok = false; break; }
            const uint32_t dst = base + x * P::kQBytes, full = bar(kShBarQFull + x);
            const int tok = w.tok0 + (w.two ? x * w.box : 0);
            mbar_arrive_expect_tx(full, static_cast<uint32_t>(w.box * a.group) * 256u);
            tma_load_3d(dst, map_q, 0, w.kvh * a.group, tok, full);
            tma_load_3d(dst + 128 * 128, map_q, 64, w.kvh * a.group, tok, full);
            pend_q |= 1u << x;
            par_q = (par_q & ~(1u << x)) | (q_phase & 1u << x);
            q_phase ^= 1u << x;
          }
          for (int j = w.k0; j < w.k1 && ok; ++j) {
            if (j > w.k0 && j * kAtKeys % kPage == 0) page = table[j * kAtKeys / kPage];
            if (page < 0 || page >= a.num_pages) {
              report_status(MDB_STATUS_BAD_PAGE);
              page = 0;
            }
            const int row = page * kPage + j * kAtKeys % kPage;
            ok = load_tile(&map_k, base + P::kOffK, kShBarKFull, kShBarKEmpty, P::kKStages, kr, pend_k, par_k, w.kvh, row) &&
                 load_tile(&map_v, base + P::kOffV, kShBarVFull, kShBarVEmpty, P::kVStages, vr, pend_v, par_v, w.kvh, row);
          }
          if (!ok) break;
        }
        if (!ok) report_status(MDB_STATUS_WAIT_TIMEOUT);
        // let the copies issued land before the CTA gives its shared memory back: another warp may have given up waiting for them
        for (int s = 0; s < P::kKStages; ++s) if (pend_k >> s & 1) mbar_wait(bar(kShBarKFull + s), par_k >> s & 1);
        for (int s = 0; s < P::kVStages; ++s) if (pend_v >> s & 1) mbar_wait(bar(kShBarVFull + s), par_v >> s & 1);
        for (int s = 0; s < 2; ++s) if (pend_q >> s & 1) mbar_wait(bar(kShBarQFull + s), par_q >> s & 1);
      }
    } else if (warp == kMmaWarp) {
      // ----------------------------------------------------------------- MMA issue (all lanes, one elected)
      // bf16 x bf16 -> fp32, M = 128, N = 128; bit 16 set: B operand MN-major
      const uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(kAtKeys >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
      const uint32_t idesc_o = idesc_s | (1u << 16);
      AtRing kr, vr;
      uint32_t p_phase = 0 /* bit 2 x + buf */, o_phase = 0, q_phase = 0 /* bit x */;
      int buf = 0;                         // score columns of the next tile of a unit of one
      bool ok = true, have = take(ok), ahead = false;
      auto wait_q = [&](int x) {
        const bool r = mbar_wait_w(bar(kShBarQFull + x), q_phase >> x & 1);
        q_phase ^= 1u << x;
        return r;
      };
      auto wait_k = [&]() {
        const bool r = mbar_wait_w(bar(kShBarKFull + kr.stage), kr.phase);
        tc_fence_after();
        return r;
      };
      auto issue_s = [&](int x, int to) {  // scores of the query tile of group x with the K tile at the ring's position
        const uint32_t q_tile = base + x * P::kQBytes, k_tile = base + P::kOffK + kr.stage * kAtTileBytes;
#pragma unroll
        for (int c = 0; c < 2; ++c)
          umma_bf16_x4_w(tmem_base + 128 * to, umma_desc_sw128(q_tile + c * (128 * 128)), 2, umma_desc_sw128(k_tile + c * kAtHalfBytes), 2, idesc_s, c);
        umma_commit_w(bar(kShBarSFull + 2 * x + to));
      };
      auto release_k = [&]() {
        umma_commit_w(bar(kShBarKEmpty + kr.stage));
        kr.advance(P::kKStages);
      };
      // O of group x (+)= P of `from` times the V tile at the ring's position
      auto issue_o = [&](int x, int from, bool first, bool last) {
        if (first) {
          // the output of the group's unit before must have been read out
          if (!mbar_wait_w(bar(kShBarOEmpty + x), (o_phase >> x & 1) ^ 1)) return false;
          o_phase ^= 1u << x;
        }
        const int i = 2 * x + from;
        const uint32_t v_tile = base + P::kOffV + vr.stage * kAtTileBytes, p = tmem_base + 128 * from, o = tmem_base + 256 + x * 128;
        if (!mbar_wait_w(bar(kShBarPFull + 2 * i), p_phase >> i & 1)) return false;
        tc_fence_after();
        umma_bf16_ts_x4_w(o, p, umma_desc_sw128_mn(v_tile), 128, idesc_o, first ? 0u : 1u);
        if (!mbar_wait_w(bar(kShBarPFull + 2 * i + 1), p_phase >> i & 1)) return false;
        p_phase ^= 1u << i;
        tc_fence_after();
        umma_bf16_ts_x4_w(o, p + 32, umma_desc_sw128_mn(v_tile + 4 * 2048), 128, idesc_o, 1u);
        umma_commit_w(bar(kShBarPDone + x));
        if (last) umma_commit_w(bar(kShBarOFull + x));
        return true;
      };
      while (ok && have) {
        if (w.two) {
          ok = wait_q(0) && wait_q(1) && wait_k();
          if (!ok) break;
          issue_s(0, 0);
          issue_s(1, 1);
          release_k();
          if (w.k1 == w.k0 + 1) { umma_commit_w(bar(kShBarQEmpty)); umma_commit_w(bar(kShBarQEmpty + 1)); }
          for (int j = w.k0; j < w.k1; ++j) {
            const bool first = j == w.k0, last = j + 1 == w.k1;
            ok = mbar_wait_w(bar(kShBarVFull + vr.stage), vr.phase) && issue_o(0, 0, first, last);
            if (!ok) break;
            if (!last) {
              ok = wait_k();
              if (!ok) break;
              issue_s(0, 0);
            }
            ok = issue_o(1, 1, first, last);
            if (!ok) break;
            umma_commit_w(bar(kShBarVEmpty + vr.stage));
            vr.advance(P::kVStages);
            if (!last) {
              issue_s(1, 1);
              release_k();
              if (j + 2 == w.k1) { umma_commit_w(bar(kShBarQEmpty)); umma_commit_w(bar(kShBarQEmpty + 1)); }
            }
          }
          have = ok && take(ok);
        } else {
          const int x = w.slot, k0 = w.k0, k1 = w.k1;
          if (!ahead) {
            ok = wait_q(x) && wait_k();
            if (!ok) break;
            issue_s(x, buf);
            release_k();
            if (k1 == k0 + 1) umma_commit_w(bar(kShBarQEmpty + x));
          }
          ahead = false;
          for (int j = k0; j < k1; ++j) {
            // the next scores first: of this unit, or of the next one where that is of one tile too
            if (j + 1 < k1) {
              ok = wait_k();
              if (!ok) break;
              issue_s(x, buf ^ 1);
              release_k();
              if (j + 2 == k1) umma_commit_w(bar(kShBarQEmpty + x));
            } else {
              have = take(ok);
              if (!ok) break;
              if (have && !w.two) {
                ok = wait_q(w.slot) && wait_k();
                if (!ok) break;
                issue_s(w.slot, buf ^ 1);
                release_k();
                if (w.k1 == w.k0 + 1) umma_commit_w(bar(kShBarQEmpty + w.slot));
                ahead = true;
              }
            }
            ok = mbar_wait_w(bar(kShBarVFull + vr.stage), vr.phase) && issue_o(x, buf, j == k0, j + 1 == k1);
            if (!ok) break;
            umma_commit_w(bar(kShBarVEmpty + vr.stage));
            vr.advance(P::kVStages);
            buf ^= 1;
          }
        }
      }
      if (!ok && lane == 0) report_status(MDB_STATUS_WAIT_TIMEOUT);
      // the products issued end before the CTA gives its memories back: this warp or another one may have given up waiting for them
      umma_commit_w(bar(kShBarEnd));
      mbar_wait_w(bar(kShBarEnd), 0);
    } else if (warp == kPartsWarp) {
      // ----------------------------------------------------------------- the CTA's parts
      ShWalk walk;
      walk.start(a);
      if (lane == 0) {
        if (blockIdx.x == 0 && a.prefix_len != nullptr && *a.prefix_len > walk.plen) report_status(MDB_STATUS_BAD_PAGE);
        for (bool more = true; more;) {
          more = walk.next(a, w);
          if (!more) w.k1 = 0;
          if (!mbar_wait(bar(kShBarPartEmpty + part.stage), part.phase ^ 1)) { report_status(MDB_STATUS_WAIT_TIMEOUT); break; }
          parts[part.stage] = w;
          mbar_arrive(bar(kShBarPartFull + part.stage));
          part.advance(P::kParts);
          if (more && w.k0 == 0) {
            a.info[w.unit] = make_int2(static_cast<int>(blockIdx.x), w.followers);
            if (w.req >= 0 && a.ctx_lens[w.req] > w.len) report_status(MDB_STATUS_BAD_PAGE);
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P::kSoftmaxRegs));
    const int x = warp >> 2;                               // group
    const int row = threadIdx.x & 127;                     // query row of the tile, and its tensor-memory lane
    const int tok_local = row / a.group;
    const uint32_t lane_field = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t o_addr = tmem_base + 256 + x * 128 + lane_field;
    const f32x2 scale = pack2(a.scale_log2, a.scale_log2);
    AtRing vr;                          // V ring position of the part's first key tile
    int buf0 = 0;                       // score columns of its first tile, in a unit of one
    uint32_t s_phase = 0 /* bit per score columns */, o_phase = 0, done_phase = 0;      // done: of the last P V
    bool ok = true;
    while (take(ok)) {
      const int tiles = w.k1 - w.k0;
      const bool mine = w.two || w.slot == x;
      if (mine) {
        const int tok = w.tok0 + (w.two ? x * w.box : 0) + tok_local;
        const bool row_valid = tok_local < w.box && tok < w.tok_end;
        const bool warp_valid = __any_sync(0xffffffffu, row_valid);
        float m_ref = -INFINITY, l = 0.f;
        for (int j = w.k0; j < w.k1; ++j) {
          const int buf = w.two ? x : (buf0 + j - w.k0) & 1;
          const uint32_t s_addr = tmem_base + 128 * buf + lane_field;
          ok = mbar_wait(bar(kShBarSFull + 2 * x + buf), s_phase >> buf & 1);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          s_phase ^= 1u << buf;
          tc_fence_after();
          const int nv = w.len - j * kAtKeys;               // keys of this tile: [0, nv)
          if (nv < kAtKeys) {
            // stale rows behind the last key must not reach O through 0 * (Inf or NaN): clear their values
            const int v_at = vr.stage + (j - w.k0), v_stage = v_at % P::kVStages;
            ok = mbar_wait(bar(kShBarVFull + v_stage), vr.phase ^ (v_at / P::kVStages & 1));
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            const int r = nv + row;
            if (r < kAtKeys) {
              const uint32_t v_row = base + P::kOffV + v_stage * kAtTileBytes + r * 128;
#pragma unroll
              for (int c = 0; c < 16; ++c)
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v_row + (c >> 3) * kAtHalfBytes + (c & 7) * 16), "r"(0u) : "memory");
            }
            fence_async_smem();
            // and their scores (NaN among them) are minus infinity: in place, where a few instructions do
            int c = nv;
            for (; c & 7; ++c) tmem_fill1(s_addr + c, -INFINITY);
            for (; c & 31; c += 8) tmem_fill8(s_addr + c, -INFINITY);
            for (; c < kAtKeys; c += 32) tmem_fill32(s_addr + c, -INFINITY);
            tmem_st_wait();
          }
          const uint32_t p_full = bar(kShBarPFull + 2 * (2 * x + buf));
          if (warp_valid) {
            float s[kAtKeys];
#pragma unroll
            for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + 32 * c, s + 32 * c);
            tmem_ld_wait();
            float mxv[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) mxv[k] = fmaxf(s[k], s[4 + k]);
#pragma unroll
            for (int c = 8; c < kAtKeys; c += 8)
#pragma unroll
              for (int k = 0; k < 4; ++k) mxv[k] = max3(mxv[k], s[c + k], s[c + 4 + k]);
            float mx = fmaxf(fmaxf(mxv[0], mxv[1]), fmaxf(mxv[2], mxv[3]));
            if (!row_valid) mx = 0.f;                             // rows that are not there hold whatever the tile held
            const float m_tile = mx * a.scale_log2;
            const bool grow = m_tile > m_ref + kAtRescaleStep || (m_ref == -INFINITY && m_tile != -INFINITY);
            if (__any_sync(0xffffffffu, grow)) {
              const float m_new = fmaxf(m_ref, m_tile);
              const float f = m_ref == -INFINITY ? 0.f : ex2_approx(m_ref - m_new);
              l *= f;
              if (j > w.k0) {
                // O is quiet once the last key tile's P V has completed (the one before completed before these scores)
                ok = mbar_wait(bar(kShBarPDone + x), done_phase ^ 1);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                  float o[32];
                  tmem_ld32(o_addr + 32 * c, o);
                  tmem_ld_wait();
#pragma unroll
                  for (int e = 0; e < 32; ++e) o[e] *= f;
                  tmem_st32(o_addr + 32 * c, o);
                }
              }
              m_ref = m_new;
            }
            // P = 2^(s * scale - m_ref) rounded to bf16 (the left operand of P V has the type of V); a masked key gives 2^-inf = 0
            const float m_use = m_ref == -INFINITY ? 0.f : m_ref;   // nothing seen yet: every s is -inf, P = 0
            const f32x2 minus = pack2(-m_use, -m_use);
            f32x2 lv[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float pk[32];                                         // 64 keys, two per word
#pragma unroll
              for (int c = 0; c < 64; c += 8) {
                float2 y[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  y[k] = unpack2(fma2(pack2(s[64 * h + c + 2 * k], s[64 * h + c + 2 * k + 1]), scale, minus));
                  y[k].x = ex2_approx(y[k].x);
                  y[k].y = ex2_approx(y[k].y);
                  lv[k] = add2(lv[k], pack2(y[k].x, y[k].y));
                  pk[(c >> 1) + k] = __uint_as_float(pack_bf16x2(y[k].x, y[k].y));
                }
              }
              tmem_st32(s_addr + 32 * h, pk);
              tmem_st_wait();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(p_full + 8 * h);
            }
            const float2 ls = unpack2(add2(add2(lv[0], lv[1]), add2(lv[2], lv[3])));
            l += ls.x + ls.y;
          } else {
            __syncwarp();
            if (lane == 0) { mbar_arrive(p_full); mbar_arrive(p_full + 8); }
          }
          done_phase ^= 1;
        }
        if (!ok) break;
        // ------------------------------------------------------------- sums of the tile
        ok = mbar_wait(bar(kShBarOFull + x), o_phase);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        o_phase ^= 1;
        tc_fence_after();
        if (warp_valid) {
          float4* po;
          float2* pm;
          int64_t stride;
          if (w.k0 > 0) {
            const int at = (w.two ? x * 128 : 0) + row;
            stride = 256;
            po = a.cont_o + static_cast<int64_t>(blockIdx.x) * 32 * 256 + at;
            pm = a.cont_ml + static_cast<int64_t>(blockIdx.x) * 256 + at;
          } else {
            const int64_t head = (w.req < 0 ? 0 : a.hkv) + w.kvh, at = static_cast<int64_t>(tok) * a.group + row % a.group;
            stride = a.rows;
            po = a.main_o + head * 32 * stride + at;
            pm = a.main_ml + head * stride + at;
          }
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float o[32];
            tmem_ld32(o_addr + 32 * c, o);
            tmem_ld_wait();
            if (row_valid) {
#pragma unroll
              for (int q4 = 0; q4 < 8; ++q4) po[(8 * c + q4) * stride] = make_float4(o[4 * q4], o[4 * q4 + 1], o[4 * q4 + 2], o[4 * q4 + 3]);
            }
          }
          if (row_valid) *pm = make_float2(m_ref, l);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kShBarOEmpty + x));
      }
      vr.phase ^= (vr.stage + tiles) / P::kVStages & 1;
      vr.stage = (vr.stage + tiles) % P::kVStages;
      if (!w.two) buf0 = (buf0 + tiles) & 1;
    }
    if (!ok && lane == 0) report_status(MDB_STATUS_WAIT_TIMEOUT);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

constexpr int kShJoin = 4;
// Joins the parts of 32 rows of a key head: prefix, CTAs that went on with it, own keys, CTAs that went on with them, in this order.  A
// lane per row, 16 channels per warp.
__global__ void __launch_bounds__(256) attn_shared_merge(const ShArgs a) {
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, quad = (threadIdx.x >> 5) * 4, kvh = blockIdx.y;
  const int at = static_cast<int>(blockIdx.x) * 32 + lane;
  const int tok = at / a.group, g = at - tok * a.group, b = tok / a.block, t = tok - b * a.block;
  pdl_wait();
  if (at >= a.rows) return;
  float m = -INFINITY, l = 0.f;
  float4 acc[4] = {};
  auto join = [&](const float2 p, const float4 (&v)[4]) {
    if (p.x == -INFINITY && p.y == p.y) return;            // (scores that are all -inf; a NaN goes on)
    const float m_new = fmaxf(m, p.x), f = ex2_approx(m - m_new), w = ex2_approx(p.x - m_new);
    m = m_new;
    l = l * f + p.y * w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc[i].x = acc[i].x * f + v[i].x * w; acc[i].y = acc[i].y * f + v[i].y * w;
      acc[i].z = acc[i].z * f + v[i].z * w; acc[i].w = acc[i].w * f + v[i].w * w;
    }
  };
  // what may be there is asked for before it is known whether it is
  float2 first_ml[2];
  float4 first[2][4];
  int2 more[2];
  int place[2], len[2];
#pragma unroll
  for (int own = 0; own < 2; ++own) {
    const int64_t head = own * a.hkv + kvh;
    first_ml[own] = a.main_ml[head * a.rows + at];
#pragma unroll
    for (int i = 0; i < 4; ++i) first[own][i] = a.main_o[(head * 32 + quad + i) * a.rows + at];
    const int box = own ? a.box_o : a.box_p, per = own ? a.per_o : a.per_p, from = own ? t : tok;
    const int tile = from / box, pair = tile / per;
    more[own] = a.info[(own ? a.hkv * (a.units_p + b * a.units_o) + kvh * a.units_o : kvh * a.units_p) + pair];
    place[own] = (tile - pair * per) * 128 + (from - tile * box) * a.group + g;
    len[own] = own ? sh_len(a, b) : sh_prefix(a);
  }
#pragma unroll
  for (int own = 0; own < 2; ++own) {
    if (len[own] == 0) continue;
    if (!sh_info_there(more[own].x, more[own].y, a.ctas)) {
      // the unit has no parts: its row is not a number
      more[own].y = 0;
      first_ml[own] = make_float2(0.f, __int_as_float(0x7fffffff));
      if (quad == 0) report_status(MDB_STATUS_WAIT_TIMEOUT);
    }
    join(first_ml[own], first[own]);
    for (int c0 = 1; c0 <= more[own].y; c0 += kShJoin) {   // several in flight
      float4 v[kShJoin][4];
      float2 ml[kShJoin];
#pragma unroll
      for (int j = 0; j < kShJoin; ++j) {
        if (c0 + j > more[own].y) break;
        const int64_t cta = more[own].x + c0 + j;
        ml[j] = a.cont_ml[cta * 256 + place[own]];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[j][i] = a.cont_o[(cta * 32 + quad + i) * 256 + place[own]];
      }
#pragma unroll
      for (int j = 0; j < kShJoin; ++j) {
        if (c0 + j > more[own].y) break;
        join(ml[j], v[j]);
      }
    }
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;             // (a NaN stays one)
  const int64_t row = static_cast<int64_t>(tok) * a.hq + kvh * a.group + g;
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    o[2 * i] = pack_bf16x2(acc[i].x * inv, acc[i].y * inv);
    o[2 * i + 1] = pack_bf16x2(acc[i].z * inv, acc[i].w * inv);
  }
  uint4* dst = reinterpret_cast<uint4*>(a.out + row * kHeadDim + quad * 4);
  dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
  dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
  if (a.lse != nullptr && quad == 0) a.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// Tiles and units of a call.
static void sh_units(ShArgs& a, int sms) {
  a.group = a.hq / a.hkv;
  a.tokens = a.bs * a.block;
  a.rows = a.tokens * a.group;
  const int most = 128 / a.group;
  a.box_p = a.tokens < most ? a.tokens : most;
  const int tiles_p = (a.tokens + a.box_p - 1) / a.box_p;
  a.box_o = a.block < most ? a.block : most;
  const int tiles_o = (a.block + a.box_o - 1) / a.box_o;
  // two tiles to a unit share the reading of the keys and the time of the products; one by one they spread over more SMs.  In key tiles
  // per SM (4.3: 23.5 us one by one, 26.5 in twos; 7: 24.6, 27.0; 14: 36.4, 36.1)
  a.per_p = tiles_p > 1 && static_cast<int64_t>(a.hkv) * tiles_p * a.prefix_pages * (kPage / kAtKeys) >= 14ll * sms ? 2 : 1;
  a.per_o = tiles_o > 1 ? 2 : 1;
  a.units_p = (tiles_p + a.per_p - 1) / a.per_p;
  a.units_o = (tiles_o + a.per_o - 1) / a.per_o;
}

}  // namespace mdb

using namespace mdb;

extern "C" {

int64_t mdb_attn_shared_workspace_bytes(int bs, int block, int hq, int hkv) {
  if (bs <= 0 || block <= 0 || hkv <= 0 || hq <= 0 || hq % hkv != 0 || hq / hkv > 128) return 0;
  const int64_t rows = static_cast<int64_t>(bs) * block * hq;
  // every row twice, 256 rows per CTA, and the units: at most one per request and head beside those of 128 rows
  return (2 * rows + 256ll * at_sm_count()) * (kHeadDim + 2) * 4 + (rows / hkv + bs + 2) * static_cast<int64_t>(hkv) * 16;
}

int mdb_attn_block_shared(const mdb_attn_shared_args* args, mdb_stream_t stream) {
  MDB_REQUIRE(args != nullptr, MDB_ERR_ARG);
  const mdb_attn_shared_args c = *args;
  MDB_REQUIRE(c.bs >= 0 && c.block > 0 && c.hq > 0 && c.hkv > 0 && c.num_pages > 0 && c.table_pages > 0 && c.prefix_pages >= 0 && c.hq % c.hkv == 0 &&
                  (c.table_stride >= c.table_pages || c.bs <= 1),
              MDB_ERR_ARG);
  if (c.bs == 0) return MDB_OK;
  MDB_REQUIRE(c.q && c.k_cache && c.v_cache && c.out && c.block_table && c.ctx_lens && (c.prefix_pages == 0 || (c.prefix_table && c.prefix_len)), MDB_ERR_ARG);
  MDB_REQUIRE(c.hq / c.hkv <= 128 && c.softmax_scale > 0.f && c.bs <= 65535 && c.block <= 65535 && c.hq <= 65535 && c.num_pages <= (1 << 23) &&
                  c.table_pages <= (1 << 22) && c.prefix_pages <= (1 << 22) && static_cast<int64_t>(c.bs) * c.block * c.hq <= (1ll << 26),
              MDB_ERR_UNSUPPORTED);
  MDB_REQUIRE(mdb_aligned16(c.q) && mdb_aligned16(c.k_cache) && mdb_aligned16(c.v_cache) && mdb_aligned16(c.out) && mdb_aligned16(c.workspace), MDB_ERR_ALIGN);
  MDB_REQUIRE(c.workspace != nullptr && c.workspace_bytes >= mdb_attn_shared_workspace_bytes(c.bs, c.block, c.hq, c.hkv), MDB_ERR_WORKSPACE);
  ShArgs a = {};
  a.out = static_cast<bf16*>(c.out);
  a.lse = c.lse;
  a.prefix_len = c.prefix_len;
  a.prefix_table = c.prefix_table;
  a.ctx_lens = c.ctx_lens;
  a.block_table = c.block_table;
  a.prefix_pages = c.prefix_pages; a.table_stride = c.table_stride; a.table_pages = c.table_pages; a.num_pages = c.num_pages;
  a.bs = c.bs; a.block = c.block; a.hq = c.hq; a.hkv = c.hkv;
  a.scale_log2 = c.softmax_scale * 1.4426950408889634f;
  const int sms = at_sm_count();
  a.ctas = sms;
  sh_units(a, sms);
  // the list's length is kept in 32 bits (2^32 is minutes of work)
  const int64_t steps = kPage / kAtKeys, most = (a.prefix_pages * steps * kShTwoStep + kShUnit) * a.units_p + (a.table_pages * steps * kShTwoStep + kShUnit) * a.units_o * a.bs;
  MDB_REQUIRE(most <= 0xf0000000ll / a.hkv, MDB_ERR_UNSUPPORTED);
  const int64_t rows = static_cast<int64_t>(a.tokens) * a.hq;
  a.main_o = static_cast<float4*>(c.workspace);
  a.cont_o = a.main_o + 2 * rows * 32;
  a.main_ml = reinterpret_cast<float2*>(a.cont_o + static_cast<int64_t>(sms) * 256 * 32);
  a.cont_ml = a.main_ml + 2 * rows;
  a.info = reinterpret_cast<int2*>(a.cont_ml + static_cast<int64_t>(sms) * 256);
  CUtensorMap map_qp, map_qo, map_k, map_v;
  if (!encode_queries(c.q, a.tokens, a.hq, a.group, a.box_p, &map_qp) ||
      (a.box_o != a.box_p && !encode_queries(c.q, a.tokens, a.hq, a.group, a.box_o, &map_qo)) ||
      !encode_cache(c.k_cache, a.num_pages, a.hkv, &map_k) || !encode_cache(c.v_cache, a.num_pages, a.hkv, &map_v))
    return MDB_ERR_CUDA;
  if (a.box_o == a.box_p) map_qo = map_qp;
  static PerDeviceOnce attr_once;
  const int dev = attr_once.slot();
  if (dev < 0) return MDB_ERR_CUDA;
  if (!attr_once.done[dev]) {
    if (cudaFuncSetAttribute(attn_shared_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ShPlan::kSmemBytes) != cudaSuccess) return MDB_ERR_CUDA;
    attr_once.done[dev] = true;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int rc = mdb_launch(attn_shared_kernel, dim3(sms), dim3(ShPlan::kThreads), ShPlan::kSmemBytes, st, map_qp, map_qo, map_k, map_v, a);
  if (rc != MDB_OK) return rc;
  return mdb_launch(attn_shared_merge, dim3((a.rows + 31) / 32, a.hkv), dim3(256), 0, st, a);
}

}  // extern "C"
