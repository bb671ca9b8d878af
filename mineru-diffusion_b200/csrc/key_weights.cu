// The attention weight every cached key has received from a block of queries, on the 5th-generation tensor cores: what eviction
// (kv_evict.cu) goes by.
//
//   out[b][h][j] = decay * previous[b][h][j] + sum over tokens t and heads g of the group of exp(q[b][t][h G + g] . k[j] * scale - lse[b][t][h G + g])
//
// lse is what the attention over all the keys returned (attention_shared.cu), so one pass over the keys is enough and no other
// statistic is needed.  The product is formed the other way round than in the attention kernels: the 128 keys of a tile are
// the rows (A operand, one key per tensor-memory lane) and the queries the columns (N = 16 .. 128), so that the sum over queries
// is a sum over one thread's registers: no exchange between threads, no atomics, one fixed order.
//
// The key tiles of all requests and heads are one list, of which every CTA takes an equal run (lengths differ and are known to
// the device alone).  Roles: a TMA warp (query tile of the run's request and head, ring of key tiles), an MMA warp, and four
// groups of four warps that take the tiles in turn.  More than 128 rows per key head go in blocks of rows over up to 16 tiles at
// a time, sums in shared memory.
//
// Bound by memory (256 bytes per key and head) up to 64 rows: 32 requests of 4096 to 8192 keys, eight heads, 73 us = 5.8 TB/s in a graph (77 in a
// long loop, at the power limit); 128 rows 82 us, 256 (twice over the keys) 76 for half the requests: exponentials, 16 a clock and SM.
// The loop over a tile's rows is kept short: with the next scores asked for ahead, in two copies of it, 5 us longer.
// A prefix's keys with the rows of a batch, 16 query and 8 key heads: 128 tokens 17 us behind 16384 keys; 1024 tokens 36 behind 1056 and 99
// behind 16384, 2048 tokens 67 and 195 (exponentials alone 4, 60, 8 and 119).  A CTA with a single tile takes all its blocks of rows through one
// group of warps, and K is loaded anew for each.
#include "mdb_common.cuh"

namespace mdb {

constexpr int kKwGroups = 4, kKwThreads = 128 * kKwGroups + 64;       // groups of four warps; TMA, MMA
constexpr int kKwMaxRows = 512 / kKwGroups;                // rows of a block: the groups' scores fill tensor memory
constexpr int kKwSegTiles = 16;                            // tiles walked at a time where there are several blocks of rows
static_assert(kKwSegTiles % kKwGroups == 0, "a group's tiles of a run");
constexpr int kKwMaxStages = 6;
constexpr int kKwSmem = 226 * 1024;

struct KwArgs {
  const float* lse;
  const float* previous;
  float* out;
  const int32_t* block_table;
  const int32_t* seqlens;
  int bs, block, hq, hkv, group, table_stride, table_pages, num_pages;
  int64_t cols;                // of out and previous
  int tokens, row_blocks;      // of a block of rows
  int n_pad, stages;
  float scale_log2, decay;
};

__device__ __forceinline__ int kw_len(const KwArgs& a, int b) {
  return static_cast<int>(max(static_cast<int64_t>(0), min(min(static_cast<int64_t>(a.seqlens[b]), a.cols), static_cast<int64_t>(a.table_pages) * kPage)));
}

// A run of tiles of one request and head.
struct KwSeg {
  int b, h, tile, tiles, len;
};
// This CTA's share of the list; every role walks it the same way.
struct KwWalk {
  int64_t left;          // tiles
  int b, off, len;       // request, tile among its heads' tiles
  __device__ __forceinline__ int tiles_of() const { return (len + kAtKeys - 1) / kAtKeys; }
  // by a whole warp
  __device__ __forceinline__ void start(const KwArgs& a) {
    const int lane = threadIdx.x & 31;
    int64_t mine = 0;
    for (int i = lane; i < a.bs; i += 32) mine += (kw_len(a, i) + kAtKeys - 1) / kAtKeys;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    const int64_t total = mine * a.hkv, G = gridDim.x, c = blockIdx.x;
    int64_t first = total * c / G;
    left = total * (c + 1) / G - first;
    b = 0; off = 0; len = 0;
    if (left == 0) return;
    for (int b0 = 0; b0 < a.bs; b0 += 32) {
      const int i = b0 + lane;
      int64_t t = i < a.bs ? static_cast<int64_t>((kw_len(a, i) + kAtKeys - 1) / kAtKeys) * a.hkv : 0, upto = t;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, first < upto);
      if (hit) {
        const int l = __ffs(hit) - 1;
        b = b0 + l;
        off = static_cast<int>(first - __shfl_sync(0xffffffffu, upto - t, l));
        break;
      }
      first -= __shfl_sync(0xffffffffu, upto, 31);
    }
    len = kw_len(a, b);
  }
  __device__ __forceinline__ bool next(const KwArgs& a, KwSeg& s) {
    if (left == 0) return false;
    int nt = tiles_of();
    while (off == nt * a.hkv) {        // (left > 0: there is a request behind this one that has tiles)
      ++b;
      off = 0;
      len = kw_len(a, b);
      nt = tiles_of();
    }
    s.b = b; s.h = off / nt; s.tile = off % nt; s.len = len;
    int64_t n = nt - s.tile;
    if (n > left) n = left;
    if (a.row_blocks > 1 && n > kKwSegTiles) n = kKwSegTiles;
    s.tiles = static_cast<int>(n);
    off += s.tiles;
    left -= s.tiles;
    return true;
  }
};

// barrier slots
enum {
  kKwBarQFull = 0, kKwBarQEmpty = 2, kKwBarSFull = 4, kKwBarSEmpty = kKwBarSFull + kKwGroups, kKwBarKFull = kKwBarSEmpty + kKwGroups,
  kKwBarKEmpty = kKwBarKFull + kKwMaxStages, kKwBarEnd = kKwBarKEmpty + kKwMaxStages /* of all products */, kKwBarCount
};

__global__ void __launch_bounds__(kKwThreads, 1)
key_weights_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const KwArgs a) {
  extern __shared__ __align__(1024) unsigned char kw_smem_raw[];
  const uint32_t raw = smem_u32(kw_smem_raw), base = (raw + 1023u) & ~1023u;
  unsigned char* gen_base = kw_smem_raw + (base - raw);
  const int q_bytes = a.n_pad * 256;                       // two channel halves of [n_pad][128 B]
  const uint32_t off_k = 2 * q_bytes, off_lse = off_k + a.stages * kAtTileBytes, off_sums = off_lse + 4 * kKwGroups * kKwMaxRows * 4;
  const uint32_t off_bars = off_sums + (a.row_blocks > 1 ? kKwSegTiles * kAtKeys * 4 : 0);
  const uint32_t bars = base + off_bars;
  auto bar = [&](int slot) { return bars + 8u * static_cast<uint32_t>(slot); };
  volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(gen_base + off_bars + 8 * kKwBarCount);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kProducerWarp = 4 * kKwGroups, kMmaWarp = kProducerWarp + 1;

  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kKwBarCount; ++s) mbar_init(bar(s), s >= kKwBarSEmpty && s < kKwBarSEmpty + kKwGroups ? 4 : 1);
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
  KwWalk walk;
  walk.start(a);
  KwSeg s;

  if (warp == kProducerWarp) {
    if (lane == 0) {
      uint32_t pend_k = 0, pend_q = 0, par_k = 0, par_q = 0;        // stages with a copy in flight, and the parity it completes
      AtRing kr, qr;
      bool ok = true;
      while (ok && walk.next(a, s)) {
        if (s.tile == 0 && a.seqlens[s.b] > s.len) report_status(MDB_STATUS_BAD_PAGE);
        for (int rb = 0; rb < a.row_blocks && ok; ++rb) {
          if (!mbar_wait(bar(kKwBarQEmpty + qr.stage), qr.phase ^ 1)) { ok = false; break; }
          const uint32_t qf = bar(kKwBarQFull + qr.stage), q_tile = base + qr.stage * q_bytes;
          mbar_arrive_expect_tx(qf, static_cast<uint32_t>(a.tokens * a.group) * 256u);
          tma_load_3d(q_tile, &map_q, 0, s.h * a.group, s.b * a.block + rb * a.tokens, qf);
          tma_load_3d(q_tile + a.n_pad * 128, &map_q, 64, s.h * a.group, s.b * a.block + rb * a.tokens, qf);
          pend_q |= 1u << qr.stage;
          par_q = (par_q & ~(1u << qr.stage)) | (qr.phase << qr.stage);
          qr.advance(2);
          for (int j = 0; j < s.tiles; ++j) {
            const int key0 = (s.tile + j) * kAtKeys;
            int page = a.block_table[static_cast<int64_t>(s.b) * a.table_stride + key0 / kPage];
            if (page < 0 || page >= a.num_pages) {
              report_status(MDB_STATUS_BAD_PAGE);
              page = 0;
            }
            if (!mbar_wait(bar(kKwBarKEmpty + kr.stage), kr.phase ^ 1)) { ok = false; break; }
            const uint32_t kf = bar(kKwBarKFull + kr.stage), k_tile = base + off_k + kr.stage * kAtTileBytes;
            mbar_arrive_expect_tx(kf, kAtTileBytes);
            tma_load_2d(k_tile, &map_k, s.h * kHeadDim, page * kPage + key0 % kPage, kf);
            tma_load_2d(k_tile + kAtHalfBytes, &map_k, s.h * kHeadDim + 64, page * kPage + key0 % kPage, kf);
            pend_k |= 1u << kr.stage;
            par_k = (par_k & ~(1u << kr.stage)) | (kr.phase << kr.stage);
            kr.advance(a.stages);
          }
        }
      }
      if (!ok) report_status(MDB_STATUS_WAIT_TIMEOUT);
      // let the copies issued land before the CTA gives its shared memory back: another warp may have given up waiting for them
      for (int i = 0; i < a.stages; ++i) if (pend_k >> i & 1) mbar_wait(bar(kKwBarKFull + i), par_k >> i & 1);
      for (int i = 0; i < 2; ++i) if (pend_q >> i & 1) mbar_wait(bar(kKwBarQFull + i), par_q >> i & 1);
    }
  } else if (warp == kMmaWarp) {
    const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(a.n_pad >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
    AtRing kr, qr;
    uint32_t s_phase = 0;              // bit per score buffer
    uint32_t seg_base = 0;
    bool ok = true;
    while (ok && walk.next(a, s)) {
      for (int rb = 0; rb < a.row_blocks && ok; ++rb) {
        if (!mbar_wait_w(bar(kKwBarQFull + qr.stage), qr.phase)) { ok = false; break; }
        const uint32_t q_tile = base + qr.stage * q_bytes;
        for (int j = 0; j < s.tiles; ++j) {
          const int buf = (seg_base + j) % kKwGroups;
          if (!mbar_wait_w(bar(kKwBarKFull + kr.stage), kr.phase) || !mbar_wait_w(bar(kKwBarSEmpty + buf), (s_phase >> buf & 1) ^ 1)) { ok = false; break; }
          s_phase ^= 1u << buf;
          tc_fence_after();
          const uint32_t k_tile = base + off_k + kr.stage * kAtTileBytes;
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_bf16_w(tmem_base + buf * kKwMaxRows, umma_desc_sw128(k_tile + (kk >> 2) * kAtHalfBytes) + 2 * (kk & 3),
                        umma_desc_sw128(q_tile + (kk >> 2) * (a.n_pad * 128)) + 2 * (kk & 3), idesc, kk > 0 ? 1u : 0u);
          umma_commit_w(bar(kKwBarKEmpty + kr.stage));
          umma_commit_w(bar(kKwBarSFull + buf));
          kr.advance(a.stages);
        }
        umma_commit_w(bar(kKwBarQEmpty + qr.stage));
        qr.advance(2);
      }
      seg_base += s.tiles;
    }
    if (!ok && lane == 0) report_status(MDB_STATUS_WAIT_TIMEOUT);
    // the products issued end before the CTA gives its memories back: this warp or another one may have given up waiting for them
    umma_commit_w(bar(kKwBarEnd));
    mbar_wait_w(bar(kKwBarEnd), 0);
  } else {
    const int wg = warp >> 2, tid = threadIdx.x & 127;     // (tid: tensor-memory lane, key of a tile)
    const uint32_t lane_field = static_cast<uint32_t>(32 * (warp & 3)) << 16;
    float* neg_lse = reinterpret_cast<float*>(gen_base + off_lse) + warp * kKwMaxRows;    // times -log2 e; a copy per warp
    float* sums = reinterpret_cast<float*>(gen_base + off_sums);
    const f32x2 scale = pack2(a.scale_log2, a.scale_log2);
    // behind the last tile of every request: no key, no weight
    for (int64_t r = blockIdx.x; r < static_cast<int64_t>(a.bs) * a.hkv; r += gridDim.x) {
      const int tiles = (kw_len(a, static_cast<int>(r / a.hkv)) + kAtKeys - 1) / kAtKeys;
      for (int64_t i = static_cast<int64_t>(tiles) * kAtKeys + threadIdx.x; i < a.cols; i += 128 * kKwGroups) a.out[r * a.cols + i] = 0.f;
    }
    uint32_t s_phase = 0, seg_base = 0;
    bool ok = true;
    while (ok && walk.next(a, s)) {
      const int64_t row = (static_cast<int64_t>(s.b) * a.hkv + s.h) * a.cols;
      for (int rb = 0; rb < a.row_blocks && ok; ++rb) {
        const int tok0 = rb * a.tokens, rows = min(a.tokens, a.block - tok0) * a.group;
        __syncwarp();
        bool none = false;             // a row that saw no key gives none a weight, whatever its query holds
        for (int r = lane; r < rows; r += 32) {
          const float l = a.lse[(static_cast<int64_t>(s.b) * a.block + tok0 + r / a.group) * a.hq + s.h * a.group + r % a.group];
          neg_lse[r] = l == -INFINITY ? -INFINITY : l * -1.4426950408889634f;
          none |= l == -INFINITY;
        }
        none = __any_sync(0xffffffffu, none);
        __syncwarp();
        for (int j = 0; j < s.tiles; ++j) {
          if (static_cast<int>((seg_base + j) % kKwGroups) != wg) continue;
          const int key = (s.tile + j) * kAtKeys + tid;
          const bool last_block = rb == a.row_blocks - 1;
          const float before = last_block && a.previous != nullptr && key < s.len ? a.previous[row + key] * a.decay : 0.f;
          ok = mbar_wait(bar(kKwBarSFull + wg), s_phase);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          s_phase ^= 1;
          tc_fence_after();
          float acc = 0.f;
          f32x2 part[4] = {0ull, 0ull, 0ull, 0ull};
          for (int c = 0; c < rows; c += 32) {
            float x[32];
            tmem_ld32(tmem_base + wg * kKwMaxRows + lane_field + c, x);      // (columns behind the last row are not looked at)
            tmem_ld_wait();
            if (none) {                // (apart: as a condition of every exponential it costs 2 %, eight rows to a key head)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (neg_lse[c + i] == -INFINITY) x[i] = 0.f;
            }
            if (c + 32 <= rows) {
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float4 n = *reinterpret_cast<const float4*>(neg_lse + c + i);
                const float2 y = unpack2(fma2(pack2(x[i], x[i + 1]), scale, pack2(n.x, n.y)));
                const float2 z = unpack2(fma2(pack2(x[i + 2], x[i + 3]), scale, pack2(n.z, n.w)));
                part[(i >> 1) & 3] = add2(part[(i >> 1) & 3], pack2(ex2_approx(y.x), ex2_approx(y.y)));
                part[((i >> 1) & 3) + 1] = add2(part[((i >> 1) & 3) + 1], pack2(ex2_approx(z.x), ex2_approx(z.y)));
              }
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c + i < rows) acc += ex2_approx(fmaf(x[i], a.scale_log2, neg_lse[c + i]));
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(kKwBarSEmpty + wg));
          const float2 p = unpack2(add2(add2(part[0], part[1]), add2(part[2], part[3])));
          acc += p.x + p.y;
          if (a.row_blocks > 1) {
            // (a place of the group's own: another group may have gone on to the next run's first block of rows)
            float& sum = sums[(wg * (kKwSegTiles / kKwGroups) + j / kKwGroups) * kAtKeys + tid];
            if (rb > 0) acc += sum;
            if (!last_block) sum = acc;
          }
          if (last_block && key < a.cols) a.out[row + key] = key < s.len ? before + acc : 0.f;
        }
      }
      seg_base += s.tiles;
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

}  // namespace mdb

using namespace mdb;

extern "C" int mdb_key_weights(const mdb_key_weights_args* args, mdb_stream_t stream) {
  MDB_REQUIRE(args != nullptr, MDB_ERR_ARG);
  const mdb_key_weights_args w = *args;
  MDB_REQUIRE(w.bs >= 0 && w.block > 0 && w.hq > 0 && w.hkv > 0 && w.num_pages > 0 && w.table_pages > 0 && w.cols > 0 && w.hq % w.hkv == 0 &&
                  (w.table_stride >= w.table_pages || w.bs <= 1),
              MDB_ERR_ARG);
  if (w.bs == 0) return MDB_OK;
  MDB_REQUIRE(w.q && w.k_cache && w.lse && w.block_table && w.ctx_lens && w.out, MDB_ERR_ARG);
  MDB_REQUIRE(mdb_aligned16(w.q) && mdb_aligned16(w.k_cache), MDB_ERR_ALIGN);
  const int group = w.hq / w.hkv;
  MDB_REQUIRE(w.bs <= 65535 && w.block <= 65535 && group <= 128 && w.num_pages <= (1 << 23) && w.table_pages <= (1 << 22) && w.cols <= (1ll << 30) &&
                  static_cast<int64_t>(w.bs) * w.block <= (1ll << 30) && w.softmax_scale > 0.f && w.hq <= 65535,
              MDB_ERR_UNSUPPORTED);
  KwArgs a = {};
  a.lse = w.lse; a.previous = w.previous; a.out = w.out;
  a.block_table = w.block_table; a.seqlens = w.ctx_lens;
  a.bs = w.bs; a.block = w.block; a.hq = w.hq; a.hkv = w.hkv; a.group = group;
  a.table_stride = w.table_stride; a.table_pages = w.table_pages; a.num_pages = w.num_pages; a.cols = w.cols;
  a.scale_log2 = w.softmax_scale * 1.4426950408889634f; a.decay = w.decay;
  a.tokens = w.block < kKwMaxRows / group ? w.block : kKwMaxRows / group;
  a.row_blocks = (w.block + a.tokens - 1) / a.tokens;
  a.n_pad = (a.tokens * group + 15) / 16 * 16;
  const int rest = 1024 + 4 * kKwGroups * kKwMaxRows * 4 + (a.row_blocks > 1 ? kKwSegTiles * kAtKeys * 4 : 0) + 8 * kKwBarCount + 16;
  a.stages = (kKwSmem - rest - 2 * a.n_pad * 256) / kAtTileBytes;
  if (a.stages > kKwMaxStages) a.stages = kKwMaxStages;
  const int smem = rest + 2 * a.n_pad * 256 + a.stages * kAtTileBytes;
  CUtensorMap map_q, map_k;
  if (!encode_queries(w.q, static_cast<int64_t>(w.bs) * w.block, w.hq, group, a.tokens, &map_q) || !encode_cache(w.k_cache, w.num_pages, w.hkv, &map_k))
    return MDB_ERR_CUDA;
  static PerDeviceOnce attr_once;
  const int dev = attr_once.slot();
  if (dev < 0) return MDB_ERR_CUDA;
  if (!attr_once.done[dev]) {
    if (cudaFuncSetAttribute(key_weights_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kKwSmem) != cudaSuccess) return MDB_ERR_CUDA;
    attr_once.done[dev] = true;
  }
  const int64_t table = static_cast<int64_t>(w.table_pages) * kPage, most = w.cols < table ? w.cols : table;
  const int64_t tiles = (most + kAtKeys - 1) / kAtKeys * w.bs * w.hkv;
  const int sms = at_sm_count();
  return mdb_launch(key_weights_kernel, dim3(tiles < sms ? static_cast<int>(tiles) : sms), dim3(kKwThreads), smem, static_cast<cudaStream_t>(stream),
                    map_q, map_k, a);
}
