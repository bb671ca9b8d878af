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
// Roles: a TMA warp (query tiles, rings of K and V tiles), an MMA warp, four softmax warps per query tile, a row per thread.
// Tensor memory: S_A (P_A) | S_B (P_B) | O_A | O_B, 128 columns each; with one tile S of even key tiles | - | O | S of odd ones.
// P goes back into the tensor memory its scores came from, in two halves, of which the first is multiplied while the second is made.
#include "mdb_common.cuh"

namespace mdb {

// Times in sixteenths of a key tile of one query tile: a key tile of one, of two, start and end of a unit; the least share of a CTA.
constexpr int kShOneStep = 16, kShTwoStep = 23, kShUnit = 32, kShMinShare = 64;

struct ShPlan {
  static constexpr int kKStages = 3, kVStages = 2;
  static constexpr int kQBytes = 2 * 128 * 128;            // a tile: two channel halves of [128 rows][128 B]
  static constexpr int kThreads = 384;                     // eight softmax warps, TMA, MMA; two idle
  static constexpr int kSoftmaxRegs = 216, kOtherRegs = 72;
  static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * 168, "registers after the split");
  static constexpr int kOffK = 2 * kQBytes;
  static constexpr int kOffV = kOffK + kKStages * kAtTileBytes;
  static constexpr int kOffBars = kOffV + kVStages * kAtTileBytes;
  static constexpr int kSmemBytes = 1024 + kOffBars + 512;
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
  int tokens;                    // bs * block
  int box_p, tiles_p, per_p, units_p;      // against the prefix: tokens of a query tile, tiles, tiles per unit, units per key head
  int box_o, tiles_o, per_o, units_o;      // against a request's own keys
  float scale_log2;
  float* main_o;                 // [2][tokens * hq][128]: prefix, own
  float* main_ml;                // [2][tokens * hq][2]: maximum in log2 units, sum
  float* cont_o;                 // [CTA][256][128]
  float* cont_ml;
  int2* info;                    // [hkv * (units_p + bs * units_o)]: CTA of the first part, how many follow
};

enum {
  kShBarQFull = 0, kShBarQEmpty = 1, kShBarKFull = 2, kShBarKEmpty = 5, kShBarVFull = 8, kShBarVEmpty = 10, kShBarSFull = 12 /* 3 */,
  kShBarPFull = 15 /* 3 x 2 halves */, kShBarPDone = 21, kShBarOFull = 23, kShBarOEmpty = 25, kShBarCount = 27
};

__device__ __forceinline__ int sh_prefix(const ShArgs& a) {
  return a.prefix_len == nullptr ? 0 : static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(*a.prefix_len), static_cast<int64_t>(a.prefix_pages) * kPage)));
}
__device__ __forceinline__ int sh_len(const ShArgs& a, int b) {
  return static_cast<int>(max(static_cast<int64_t>(0), min(static_cast<int64_t>(a.ctx_lens[b]), static_cast<int64_t>(a.table_pages) * kPage)));
}
__device__ __forceinline__ int sh_steps(int len) { return len / kAtKeys + (len % kAtKeys != 0); }
__device__ __forceinline__ int64_t sh_cost(int steps, int per) {
  return steps == 0 ? 0 : static_cast<int64_t>(steps) * (per == 2 ? kShTwoStep : kShOneStep) + kShUnit;
}

// A part of a unit.
struct ShPart {
  int req;                 // -1: the prefix
  int kvh, unit;           // unit: its place in info
  int tok0, tok1;          // first tokens of tile A and B (of all requests' tokens); tile B is there where `two`
  bool two;
  int tok_end;             // the rows end here
  int box;                 // tokens of a tile
  int len, k0, k1, steps;  // keys of the unit; key tiles of the part, of the unit
};

// A CTA's run of the list; every role walks it the same way.
struct ShWalk {
  int64_t x0, x1, total, at;     // run, length of the list, start of the unit at the cursor
  int share;                     // CTAs that have a run
  int plen, len;                 // of the prefix, of the request at the cursor
  int b, u;                      // cursor: request (-1: prefix), unit among its key heads' units
  // by a whole warp
  __device__ __forceinline__ void start(const ShArgs& a) {
    const int lane = threadIdx.x & 31;
    plen = sh_prefix(a);
    int64_t own = 0;
    for (int i = lane; i < a.bs; i += 32) own += sh_cost(sh_steps(sh_len(a, i)), a.per_o);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) own += __shfl_xor_sync(0xffffffffu, own, o);
    const int64_t cost_p = sh_cost(sh_steps(plen), a.per_p), all_p = cost_p * a.hkv * a.units_p, per_req = static_cast<int64_t>(a.hkv) * a.units_o;
    total = all_p + own * per_req;
    share = static_cast<int>(min(static_cast<int64_t>(gridDim.x), max(static_cast<int64_t>(1), total / kShMinShare)));
    const int c = static_cast<int>(blockIdx.x);
    x0 = x1 = at = 0;
    b = -1; u = 0; len = 0;
    if (c >= share) return;
    x0 = total * c / share;
    x1 = total * (c + 1) / share;
    if (x0 < all_p) {
      u = static_cast<int>(x0 / cost_p);
      at = u * cost_p;
      return;
    }
    at = all_p;
    for (int b0 = 0; b0 < a.bs; b0 += 32) {
      const int i = b0 + lane;
      const int64_t mine = i < a.bs ? sh_cost(sh_steps(sh_len(a, i)), a.per_o) * per_req : 0;
      int64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, x0 < at + upto);
      if (hit) {
        const int l = __ffs(hit) - 1;
        b = b0 + l;
        at += __shfl_sync(0xffffffffu, upto - mine, l);
        const int64_t each = __shfl_sync(0xffffffffu, mine, l) / per_req;
        u = static_cast<int>((x0 - at) / each);
        at += u * each;
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
      const int units = prefix ? a.units_p : a.units_o, per = prefix ? a.per_p : a.per_o;
      const int n = prefix ? plen : len, steps = sh_steps(n);
      if (steps == 0 || u == a.hkv * units) {              // behind the units of the prefix or of a request
        ++b;
        u = 0;
        if (b >= a.bs) return false;
        len = sh_len(a, b);
        continue;
      }
      const int64_t cost = sh_cost(steps, per);
      p.k0 = x0 <= at ? 0 : static_cast<int>((x0 - at) * steps / cost);
      p.k1 = x1 >= at + cost ? steps : static_cast<int>((x1 - at) * steps / cost);
      p.req = b;
      p.kvh = u / units;
      p.unit = prefix ? u : a.hkv * (a.units_p + b * a.units_o) + u;
      p.box = prefix ? a.box_p : a.box_o;
      const int first = (u % units) * per;
      p.tok0 = (prefix ? 0 : b * a.block) + first * p.box;
      p.tok1 = p.tok0 + p.box;
      p.tok_end = prefix ? a.tokens : (b + 1) * a.block;
      p.two = per == 2 && p.tok1 < p.tok_end;
      p.len = n; p.steps = steps;
      at += cost;
      ++u;
      if (p.k1 > p.k0) return true;
    }
    return false;
  }
  // how many CTAs behind this one have a part of the unit that `next` gave last
  __device__ __forceinline__ int followers(const ShArgs& a, const ShPart& p) const {
    const int64_t cost = sh_cost(p.steps, p.req < 0 ? a.per_p : a.per_o), s = at - cost;
    int n = 0;
    for (int c = static_cast<int>(blockIdx.x) + 1; c < share; ++c, ++n) {
      const int64_t x = total * c / share;
      if (x >= at || (x - s) * p.steps / cost >= p.steps) break;
    }
    return n;
  }
};

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t sh_score_col(int buf) { return buf == 2 ? 384u : 128u * buf; }

__global__ void __launch_bounds__(ShPlan::kThreads, 1)
attn_shared_kernel(const __grid_constant__ CUtensorMap map_qp, const __grid_constant__ CUtensorMap map_qo, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const ShArgs a) {
  using P = ShPlan;
  constexpr int kProducerWarp = 8, kMmaWarp = 9;
  extern __shared__ __align__(1024) unsigned char sh_smem_raw[];
  const uint32_t raw = smem_u32(sh_smem_raw), base = (raw + 1023u) & ~1023u;
  unsigned char* gen_base = sh_smem_raw + (base - raw);
  const uint32_t bars = base + P::kOffBars;
  auto bar = [&](int slot) { return bars + 8u * static_cast<uint32_t>(slot); };
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(gen_base + P::kOffBars + 8 * kShBarCount);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kShBarCount; ++s) mbar_init(bar(s), (s >= kShBarPFull && s < kShBarPFull + 6) || s >= kShBarOEmpty ? 4 : 1);
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
  ShWalk walk;
  walk.start(a);
  ShPart w;

  if (warp >= kProducerWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P::kOtherRegs));
    if (warp == kProducerWarp) {
      // ------------------------------------------------------------------ producer
      if (lane == 0) {
        AtRing kr, vr;
        uint32_t q_phase = 0;
        uint32_t pend_k = 0, pend_v = 0, pend_q = 0;          // stages with a copy in flight, and the parity it completes
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
        if (blockIdx.x == 0 && a.prefix_len != nullptr && *a.prefix_len > walk.plen) report_status(MDB_STATUS_BAD_PAGE);
        while (ok && walk.next(a, w)) {
          if (w.req >= 0 && w.k0 == 0 && a.ctx_lens[w.req] > w.len) report_status(MDB_STATUS_BAD_PAGE);
          if (!mbar_wait(bar(kShBarQEmpty), q_phase ^ 1)) { ok = false; break; }
          const CUtensorMap* map_q = w.req < 0 ? &map_qp : &map_qo;
          mbar_arrive_expect_tx(bar(kShBarQFull), static_cast<uint32_t>(w.box * a.group) * 256u * (w.two ? 2u : 1u));
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (x == 1 && !w.two) break;
            const uint32_t dst = base + x * P::kQBytes;
            const int tok = x == 0 ? w.tok0 : w.tok1;
            tma_load_3d(dst, map_q, 0, w.kvh * a.group, tok, bar(kShBarQFull));
            tma_load_3d(dst + 128 * 128, map_q, 64, w.kvh * a.group, tok, bar(kShBarQFull));
          }
          pend_q = 1u;
          par_q = q_phase;
          q_phase ^= 1;
          const int32_t* table = w.req < 0 ? a.prefix_table : a.block_table + static_cast<int64_t>(w.req) * a.table_stride;
          for (int j = w.k0; j < w.k1 && ok; ++j) {
            int page = table[j * kAtKeys / kPage];
            if (page < 0 || page >= a.num_pages) {
              report_status(MDB_STATUS_BAD_PAGE);
              page = 0;
            }
            const int row = page * kPage + j * kAtKeys % kPage;
            ok = load_tile(&map_k, base + P::kOffK, kShBarKFull, kShBarKEmpty, P::kKStages, kr, pend_k, par_k, w.kvh, row) &&
                 load_tile(&map_v, base + P::kOffV, kShBarVFull, kShBarVEmpty, P::kVStages, vr, pend_v, par_v, w.kvh, row);
          }
        }
        if (!ok) {
          report_status(MDB_STATUS_WAIT_TIMEOUT);
          // let the copies already issued land before the CTA gives its shared memory back
          for (int s = 0; s < P::kKStages; ++s) if (pend_k >> s & 1) mbar_wait(bar(kShBarKFull + s), par_k >> s & 1);
          for (int s = 0; s < P::kVStages; ++s) if (pend_v >> s & 1) mbar_wait(bar(kShBarVFull + s), par_v >> s & 1);
          if (pend_q) mbar_wait(bar(kShBarQFull), par_q);
        }
      }
    } else if (warp == kMmaWarp) {
      // ----------------------------------------------------------------- MMA issue (all lanes, one elected)
      // bf16 x bf16 -> fp32, M = 128, N = 128; bit 16 set: B operand MN-major
      const uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(kAtKeys >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
      const uint32_t idesc_o = idesc_s | (1u << 16);
      AtRing kr, vr;
      uint32_t p_phase = 0 /* bit per score buffer */, o_phase[2] = {0, 0}, q_phase = 0;
      bool ok = true;
      while (ok && walk.next(a, w)) {
        const bool alone = !w.two;
        if (!mbar_wait_w(bar(kShBarQFull), q_phase)) { ok = false; break; }
        q_phase ^= 1;
        auto issue_s = [&](int x, int buf) {           // scores of tile x with the K tile at the ring's position
          const uint32_t q_tile = base + x * P::kQBytes, k_tile = base + P::kOffK + kr.stage * kAtTileBytes;
#pragma unroll
          for (int c = 0; c < 2; ++c)
            umma_bf16_x4_w(tmem_base + sh_score_col(buf), umma_desc_sw128(q_tile + c * (128 * 128)), 2, umma_desc_sw128(k_tile + c * kAtHalfBytes), 2, idesc_s, c);
          umma_commit_w(bar(kShBarSFull + buf));
        };
        auto release_k = [&](int j) {
          umma_commit_w(bar(kShBarKEmpty + kr.stage));
          kr.advance(P::kKStages);
          if (j == w.k1 - 1) umma_commit_w(bar(kShBarQEmpty));
        };
        if (!mbar_wait_w(bar(kShBarKFull + kr.stage), kr.phase)) { ok = false; break; }
        tc_fence_after();
        issue_s(0, 0);
        if (w.two) issue_s(1, 1);
        release_k(w.k0);
        for (int j = w.k0; j < w.k1 && ok; ++j) {
          const bool more = j + 1 < w.k1;
          const int odd = (j - w.k0) & 1;
          bool k_there = false;
          if (alone && more) {
            // the other buffer held the last key tile, whose P V has been issued; or an output of tile B that must have been read out
            if (j == w.k0 && !mbar_wait_w(bar(kShBarOEmpty + 1), o_phase[1] ^ 1)) { ok = false; break; }
            if (!mbar_wait_w(bar(kShBarKFull + kr.stage), kr.phase)) { ok = false; break; }
            tc_fence_after();
            issue_s(0, odd ? 0 : 2);
            release_k(j + 1);
          }
          if (!mbar_wait_w(bar(kShBarVFull + vr.stage), vr.phase)) { ok = false; break; }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (x == 1 && alone) break;
            const int buf = alone && odd ? 2 : x;
            if (j == w.k0) {
              // the previous unit's accumulator must have been read out
              if (!mbar_wait_w(bar(kShBarOEmpty + x), o_phase[x] ^ 1)) { ok = false; break; }
              o_phase[x] ^= 1;
            }
            const uint32_t v_tile = base + P::kOffV + vr.stage * kAtTileBytes, p = tmem_base + sh_score_col(buf), o = tmem_base + 256 + x * 128;
            if (!mbar_wait_w(bar(kShBarPFull + 2 * buf), p_phase >> buf & 1)) { ok = false; break; }
            tc_fence_after();
            umma_bf16_ts_x4_w(o, p, umma_desc_sw128_mn(v_tile), 128, idesc_o, j > w.k0 ? 1u : 0u);
            if (!mbar_wait_w(bar(kShBarPFull + 2 * buf + 1), p_phase >> buf & 1)) { ok = false; break; }
            p_phase ^= 1u << buf;
            tc_fence_after();
            umma_bf16_ts_x4_w(o, p + 32, umma_desc_sw128_mn(v_tile + 4 * 2048), 128, idesc_o, 1u);
            umma_commit_w(bar(kShBarPDone + x));
            if (!more) umma_commit_w(bar(kShBarOFull + x));
            if (!alone && more) {
              if (!k_there && !mbar_wait_w(bar(kShBarKFull + kr.stage), kr.phase)) { ok = false; break; }
              k_there = true;
              tc_fence_after();
              issue_s(x, x);
            }
          }
          if (!ok) break;
          umma_commit_w(bar(kShBarVEmpty + vr.stage));
          vr.advance(P::kVStages);
          if (!alone && more) release_k(j + 1);
        }
      }
      if (!ok && lane == 0) report_status(MDB_STATUS_WAIT_TIMEOUT);
    }
  } else {
    // ------------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P::kSoftmaxRegs));
    const int x = warp >> 2;                               // tile A or B
    const int row = threadIdx.x & 127;                     // query row of the tile, and its tensor-memory lane
    const int tok_local = row / a.group, head_in_group = row % a.group;
    const uint32_t lane_field = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    const uint32_t o_addr = tmem_base + 256 + x * 128 + lane_field;
    const f32x2 scale = pack2(a.scale_log2, a.scale_log2);
    AtRing vr;                          // V ring position of the part's first key tile
    uint32_t s_phase = 0 /* bit per buffer */, o_phase = 0, done_phase = 0;      // done: of the last P V
    bool ok = true;
    while (ok && walk.next(a, w)) {
      const int tiles = w.k1 - w.k0;
      if (x == 0 && threadIdx.x == 0 && w.k0 == 0) a.info[w.unit] = make_int2(static_cast<int>(blockIdx.x), walk.followers(a, w));
      auto skip_v = [&]() { vr.phase ^= (vr.stage + tiles) / P::kVStages & 1; vr.stage = (vr.stage + tiles) % P::kVStages; };
      if (x == 1 && !w.two) {
        skip_v();
        continue;
      }
      const int tok = (x == 0 ? w.tok0 : w.tok1) + tok_local;
      const bool row_valid = tok_local < w.box && tok < w.tok_end;
      const bool warp_valid = __any_sync(0xffffffffu, row_valid);
      float m_ref = -INFINITY, l = 0.f;
      for (int j = w.k0; j < w.k1; ++j) {
        const int odd = (j - w.k0) & 1, buf = !w.two && odd ? 2 : x;
        const uint32_t s_addr = tmem_base + sh_score_col(buf) + lane_field;
        ok = mbar_wait(bar(kShBarSFull + buf), s_phase >> buf & 1);
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
        }
        if (warp_valid) {
          float s[kAtKeys];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + 32 * c, s + 32 * c);
          tmem_ld_wait();
          if (nv < kAtKeys) {
#pragma unroll
            for (int c = 0; c < kAtKeys; ++c) if (c >= nv) s[c] = -INFINITY;   // also replaces NaN from stale rows
          }
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
            if (lane == 0) mbar_arrive(bar(kShBarPFull + 2 * buf + h));
          }
          const float2 ls = unpack2(add2(add2(lv[0], lv[1]), add2(lv[2], lv[3])));
          l += ls.x + ls.y;
        } else {
          __syncwarp();
          if (lane == 0) { mbar_arrive(bar(kShBarPFull + 2 * buf)); mbar_arrive(bar(kShBarPFull + 2 * buf + 1)); }
        }
        done_phase ^= 1;
      }
      if (!ok) break;
      skip_v();
      // ------------------------------------------------------------- sums of the tile
      ok = mbar_wait(bar(kShBarOFull + x), o_phase);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      o_phase ^= 1;
      tc_fence_after();
      if (warp_valid) {
        const int64_t rows = static_cast<int64_t>(a.tokens) * a.hq;
        const int64_t at = w.k0 > 0 ? static_cast<int64_t>(blockIdx.x) * 256 + x * 128 + row
                                    : (w.req < 0 ? 0 : rows) + static_cast<int64_t>(tok) * a.hq + w.kvh * a.group + head_in_group;
        float4* po = reinterpret_cast<float4*>((w.k0 > 0 ? a.cont_o : a.main_o) + at * kHeadDim);
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float o[32];
          tmem_ld32(o_addr + 32 * c, o);
          tmem_ld_wait();
          if (row_valid) {
#pragma unroll
            for (int q4 = 0; q4 < 8; ++q4) po[8 * c + q4] = make_float4(o[4 * q4], o[4 * q4 + 1], o[4 * q4 + 2], o[4 * q4 + 3]);
          }
        }
        if (row_valid) *reinterpret_cast<float2*>((w.k0 > 0 ? a.cont_ml : a.main_ml) + at * 2) = make_float2(m_ref, l);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kShBarOEmpty + x));
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

// Joins a row's parts: prefix, CTAs that went on with it, own keys, CTAs that went on with them, in this order; a warp per row.
__global__ void __launch_bounds__(256) attn_shared_merge(const ShArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t rows = static_cast<int64_t>(a.tokens) * a.hq, r = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r >= rows) return;
  const int tok = static_cast<int>(r / a.hq), head = static_cast<int>(r % a.hq), kvh = head / a.group, g = head % a.group;
  const int b = tok / a.block, t = tok % a.block;
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto join = [&](const float* o, const float* ml, int64_t at) {
    const float2 p = *reinterpret_cast<const float2*>(ml + at * 2);
    const float4 v = *reinterpret_cast<const float4*>(o + at * kHeadDim + lane * 4);
    if (p.x == -INFINITY) return;                          // (scores that are all -inf)
    const float m_new = fmaxf(m, p.x), f = ex2_approx(m - m_new), w = ex2_approx(p.x - m_new);
    m = m_new;
    l = l * f + p.y * w;
    acc.x = acc.x * f + v.x * w; acc.y = acc.y * f + v.y * w; acc.z = acc.z * f + v.z * w; acc.w = acc.w * f + v.w * w;
  };
#pragma unroll
  for (int own = 0; own < 2; ++own) {
    const int len = own ? sh_len(a, b) : sh_prefix(a);
    if (len == 0) continue;
    const int box = own ? a.box_o : a.box_p, per = own ? a.per_o : a.per_p, units = own ? a.units_o : a.units_p;
    const int at = own ? t : tok, tile = at / box;
    const int unit = (own ? a.hkv * (a.units_p + b * a.units_o) : 0) + kvh * units + tile / per;
    const int2 more = a.info[unit];
    join(a.main_o, a.main_ml, (own ? rows : 0) + r);
    const int64_t place = static_cast<int64_t>(tile % per) * 128 + (at % box) * a.group + g;
    for (int c = 1; c <= more.y; ++c) join(a.cont_o, a.cont_ml, static_cast<int64_t>(more.x + c) * 256 + place);
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;             // (a NaN stays one)
  *reinterpret_cast<uint2*>(a.out + r * kHeadDim + lane * 4) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  if (a.lse != nullptr && lane == 0) a.lse[r] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// Tiles and units of a call.
static void sh_units(ShArgs& a) {
  a.group = a.hq / a.hkv;
  a.tokens = a.bs * a.block;
  const int most = 128 / a.group;
  a.box_p = a.tokens < most ? a.tokens : most;
  a.tiles_p = (a.tokens + a.box_p - 1) / a.box_p;
  a.box_o = a.block < most ? a.block : most;
  a.tiles_o = (a.block + a.box_o - 1) / a.box_o;
  a.per_p = a.tiles_p > 1 ? 2 : 1;
  a.per_o = a.tiles_o > 1 ? 2 : 1;
  a.units_p = (a.tiles_p + a.per_p - 1) / a.per_p;
  a.units_o = (a.tiles_o + a.per_o - 1) / a.per_o;
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

int mdb_attn_block_shared(const void* q, const void* k_cache, const void* v_cache, void* out, float* lse, const int32_t* prefix_table,
                          int prefix_pages, const int32_t* prefix_len, const int32_t* block_table, int table_stride, int table_pages, const int32_t* ctx_lens, int bs,
                          int block, int hq, int hkv, int num_pages, float softmax_scale, void* workspace, int64_t workspace_bytes, mdb_stream_t stream) {
  MDB_REQUIRE(bs >= 0 && block > 0 && hq > 0 && hkv > 0 && num_pages > 0 && table_pages > 0 && (table_stride >= table_pages || bs <= 1) && prefix_pages >= 0 && hq % hkv == 0, MDB_ERR_ARG);
  if (bs == 0) return MDB_OK;
  MDB_REQUIRE(q && k_cache && v_cache && out && block_table && ctx_lens && (prefix_pages == 0 || (prefix_table && prefix_len)), MDB_ERR_ARG);
  MDB_REQUIRE(hq / hkv <= 128 && softmax_scale > 0.f && bs <= 65535 && block <= 65535 && hq <= 65535 && num_pages <= (1 << 23) &&
                  table_pages <= (1 << 22) && prefix_pages <= (1 << 22) && static_cast<int64_t>(bs) * block * hq <= (1ll << 30),
              MDB_ERR_UNSUPPORTED);
  MDB_REQUIRE(mdb_aligned16(q) && mdb_aligned16(k_cache) && mdb_aligned16(v_cache) && mdb_aligned16(out) && mdb_aligned16(workspace), MDB_ERR_ALIGN);
  MDB_REQUIRE(workspace != nullptr && workspace_bytes >= mdb_attn_shared_workspace_bytes(bs, block, hq, hkv), MDB_ERR_WORKSPACE);
  ShArgs a = {};
  a.out = static_cast<bf16*>(out);
  a.lse = lse;
  a.prefix_len = prefix_pages > 0 ? prefix_len : nullptr;
  a.prefix_table = prefix_table;
  a.ctx_lens = ctx_lens;
  a.block_table = block_table;
  a.prefix_pages = prefix_pages; a.table_stride = table_stride; a.table_pages = table_pages; a.num_pages = num_pages;
  a.bs = bs; a.block = block; a.hq = hq; a.hkv = hkv;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  sh_units(a);
  const int sms = at_sm_count();
  const int64_t rows = static_cast<int64_t>(a.tokens) * hq;
  a.main_o = static_cast<float*>(workspace);
  a.cont_o = a.main_o + 2 * rows * kHeadDim;
  a.main_ml = a.cont_o + static_cast<int64_t>(sms) * 256 * kHeadDim;
  a.cont_ml = a.main_ml + 2 * rows * 2;
  a.info = reinterpret_cast<int2*>(a.cont_ml + static_cast<int64_t>(sms) * 256 * 2);
  CUtensorMap map_qp, map_qo, map_k, map_v;
  if (!encode_queries(q, a.tokens, hq, a.group, a.box_p, &map_qp) || !encode_queries(q, a.tokens, hq, a.group, a.box_o, &map_qo) ||
      !encode_cache(k_cache, num_pages, hkv, &map_k) || !encode_cache(v_cache, num_pages, hkv, &map_v))
    return MDB_ERR_CUDA;
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
  return mdb_launch(attn_shared_merge, dim3(static_cast<unsigned>((rows + 7) / 8)), dim3(256), 0, st, a);
}

}  // extern "C"
