// Eviction from the paged cache by the weight its keys have received (key_weights.cu).
//
// Per request and key head: of n keys the last `recent` stay, and of those in front the budget - recent with the largest weight
// (NaN counts as the lowest, the lowest index wins a tie).  The rows that stay are packed, in order, into the first places of the
// request's pages, or of other pages; their weights move with them.
//
//   evict_select_kernel   a CTA per (request, key head).  Radix selection over the weights' bits in order (11, 11 and 10 bits, counts in
//                         shared memory): after it the key of the last one that stays is known, and how many of its equals do.
//                         Then the places in order, from sums over the CTA.  Up to 32768 weights stay in registers, 32 a thread.
//   evict_move_kernel     rows of K and V, a row's places looked up once for all its pieces.  To other pages: any order, 256 rows per
//                         CTA, all heads of a stretch of tokens side by side (they lie side by side in memory).  In place a row's
//                         new place is never behind its old one, so a CTA that has a slice of the channels of all rows walks
//                         them in order, loads of a step in front of its stores.
//
// Bound by memory: rows read and written once.  16 requests of 16384 to 32768 keys, eight heads, 8192 stay: 170 us = 6.3 TB/s for the
// rows (places looked up by every piece, heads one behind the other: 297), 22 us for the selection in front of them (31 before its
// weights stayed in registers); 189 together.  In place 16 requests of 32768 keys take 225 us and one of 30000 that keeps 8000 takes 48
// (20 of them the selection, with a CTA per key head) for 10 of reading and writing: a CTA walks its slice alone, a step at a time.
#include "mdb_common.cuh"

namespace mdb {

constexpr int kEvThreads = 1024, kEvQuads = 8, kEvStride = 4 * kEvThreads, kEvPage = kEvQuads * kEvStride;
constexpr int kEvBins = 2048;
constexpr int kEvMoveThreads = 256, kEvMovePieces = 8;     // pieces of 16 bytes in flight per thread
// rows of a CTA, or of a step in place (256: 63 for 50 us, one request of 30000 keys that keeps 8000)
constexpr int kEvMoveRows = 256, kEvStepRows = 1024;

__device__ __forceinline__ bool mdb_device_aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// Bits that order like the numbers: negative ones upside down, -0 as 0, NaN lowest; and the number back.
__device__ __forceinline__ uint32_t ev_key(float w) {
  const uint32_t b = __float_as_uint(w + 0.0f);
  const uint32_t k = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
  return w != w ? 0u : k;
}
__device__ __forceinline__ float ev_number(uint32_t k) {
  return __uint_as_float(k ^ (static_cast<uint32_t>(static_cast<int32_t>(~k) >> 31) | 0x80000000u));
}

// Sum over the threads in front of this one, and of all, over the CTA.
__device__ __forceinline__ uint32_t ev_before(uint32_t mine, uint32_t* warp_sums, uint32_t& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += up;
  }
  if (lane == 31) warp_sums[warp] = upto;
  __syncthreads();
  const uint32_t w = warp_sums[lane];                      // 32 warps
  const uint32_t in_front = __reduce_add_sync(0xffffffffu, lane < warp ? w : 0u);
  all = __reduce_add_sync(0xffffffffu, w);
  return in_front + upto - mine;
}

// Keys of weights [base, base + kEvPage) of the `front` ones, four neighbours at a time: k[4 q + c] is number base + q kEvStride + 4 tid
// + c.  0, the lowest, behind the last: such a one counts among the lowest and lies behind all of them, so it never stays.
__device__ __forceinline__ void ev_load(const float* w, int base, int front, bool wide, uint32_t (&k)[4 * kEvQuads]) {
  const int i0 = base + 4 * static_cast<int>(threadIdx.x);
  // all loads first: one trip to memory, not one for every four
#pragma unroll
  for (int q = 0; q < kEvQuads; ++q) {
    const int i = i0 + q * kEvStride;
    if (wide && i + 3 < front) {
      const uint4 v = *reinterpret_cast<const uint4*>(w + i);
      k[4 * q] = v.x; k[4 * q + 1] = v.y; k[4 * q + 2] = v.z; k[4 * q + 3] = v.w;
    }
  }
#pragma unroll
  for (int q = 0; q < kEvQuads; ++q) {
    if (base + q * kEvStride >= front) break;
    const int i = i0 + q * kEvStride;
    const bool there = wide && i + 3 < front;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (!there) k[4 * q + c] = i + c < front ? __float_as_uint(w[i + c]) : 0x7fffffffu;      // (a NaN: 0)
      k[4 * q + c] = ev_key(__uint_as_float(k[4 * q + c]));
    }
  }
}

// out_cols: of weights_out; apart: the rows go to other pages, in any order.
__global__ void __launch_bounds__(kEvThreads, 1) evict_select_kernel(const mdb_kv_evict_args a, const int64_t out_cols, const bool apart) {
  __shared__ uint32_t counts[kEvBins];
  __shared__ uint32_t warp_sums[2][32];
  __shared__ uint32_t quad_sums[kEvQuads * 32];
  __shared__ uint32_t found[2];
  const int b = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_launch_dependents();
  for (int i = tid; i < kEvBins; i += kEvThreads) counts[i] = 0;
  pdl_wait();
  int n = a.seqlens[b];
  const int64_t most = min(static_cast<int64_t>(a.table_pages) * kPage, static_cast<int64_t>(a.weight_cols));
  if (n > most) {
    n = static_cast<int>(most);
    if (tid == 0) report_status(MDB_STATUS_BAD_PAGE);
  }
  n = max(n, 0);
  const float* w = a.weights + b * a.weight_row + h * a.weight_head;
  const bool wide = mdb_device_aligned16(w);
  int32_t* kept = a.kept + (static_cast<int64_t>(b) * a.kv_heads + h) * a.budget;
  float* w_out = a.weights_out == nullptr ? nullptr : a.weights_out + b * a.weight_out_row + h * a.weight_out_head;
  // of n keys in front of the recent ones, `need` stay
  const int recent = n > a.budget ? a.recent : n, front = n - recent, need = n > a.budget ? a.budget - recent : 0;
  if (need > 0) {
    uint32_t last = 0, left = need;                        // key of the last one that stays; how many of its equals do
    uint32_t k[4 * kEvQuads];
    ev_load(w, 0, front, wide, k);
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      constexpr int kShift[3] = {21, 10, 0};
      const int shift = kShift[pass], bins = pass == 2 ? 1024 : 2048;
      __syncthreads();                                     // the counts are zero
      for (int base = 0; base < front; base += kEvPage) {
        if (front > kEvPage && (base > 0 || pass > 0)) ev_load(w, base, front, wide, k);
#pragma unroll
        for (int q = 0; q < kEvQuads; ++q) {
          if (base + q * kEvStride >= front) break;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t u = k[4 * q + c];
            if (pass == 0 || (u ^ last) >> (pass == 1 ? 21 : 10) == 0) atomicAdd(&counts[(u >> shift) & (bins - 1)], 1u);
          }
        }
      }
      __syncthreads();
      // the bin, from the highest on, in which the left-th key lies: two bins per thread, highest first
      const int hi = bins - 1 - 2 * tid;
      const uint32_t c0 = hi >= 0 ? counts[hi] : 0u, c1 = hi >= 0 ? counts[hi - 1] : 0u;
      if (hi >= 0) { counts[hi] = 0; counts[hi - 1] = 0; }
      uint32_t all;
      const uint32_t in_front = ev_before(c0 + c1, warp_sums[pass & 1], all);
      if (in_front < left && left <= in_front + c0 + c1) {
        const bool second = left > in_front + c0;
        found[0] = static_cast<uint32_t>(second ? hi - 1 : hi);
        found[1] = left - in_front - (second ? c0 : 0u);
      }
      __syncthreads();
      last |= found[0] << shift;
      left = found[1];
    }
    const uint32_t equals = left;
    // places in order; all of a page is read before any of its places is written (weights_out may be weights)
    uint32_t done = 0, done_equals = 0;
    for (int base = 0; base < front; base += kEvPage) {
      if (front > kEvPage) ev_load(w, base, front, wide, k);
      uint32_t above = 0, same = 0, before[kEvQuads];      // a bit per key; counts in front within the warp: above | equals << 16
#pragma unroll
      for (int q = 0; q < kEvQuads; ++q) {
        if (base + q * kEvStride >= front) break;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          above |= static_cast<uint32_t>(k[4 * q + c] > last) << (4 * q + c);
          same |= static_cast<uint32_t>(k[4 * q + c] == last) << (4 * q + c);
        }
        const uint32_t mine = __popc(above >> (4 * q)) | __popc(same >> (4 * q)) << 16;
        uint32_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += up;
        }
        before[q] = upto - mine;
        if (lane == 31) quad_sums[q * 32 + warp] = upto;
      }
      __syncthreads();
      // (a page has up to 2^15 of either kind: 16 bits each)
      if (warp < kEvQuads && base + warp * kEvStride < front) {
        const uint32_t mine = quad_sums[tid];
        uint32_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += up;
        }
        quad_sums[tid] = upto - mine;
        if (lane == 31) warp_sums[0][warp] = upto;
      }
      __syncthreads();
      uint32_t page = 0;
#pragma unroll
      for (int q = 0; q < kEvQuads; ++q) {
        if (base + q * kEvStride >= front) break;
        const uint32_t in_front = page + quad_sums[q * 32 + warp] + before[q];
        page += warp_sums[0][q];
        uint32_t ties = done_equals + (in_front >> 16), keep = above >> (4 * q) & 15u;
        const uint32_t at = done + (in_front & 0xffffu) + min(ties, equals), tied = same >> (4 * q) & 15u;
        if (tied) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (tied >> c & 1) keep |= static_cast<uint32_t>(ties++ < equals) << c;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t to = at + __popc(keep & ((1u << c) - 1u));
          if (keep >> c & 1) {
            kept[to] = base + q * kEvStride + 4 * tid + c;
            if (w_out != nullptr) w_out[to] = ev_number(k[4 * q + c]);
          }
        }
      }
      done += page & 0xffffu;
      done_equals += page >> 16;
      __syncthreads();
    }
  }
  float y = tid < recent && w_out != nullptr ? w[front + tid] : 0.f;
  // does the request write a page that it reads?  (looked up here, under the first of these loads: in front of the selection 1 us longer)
  bool both = false;
  if (apart) {
    const int32_t* from = a.block_table + static_cast<int64_t>(b) * a.table_stride;
    const int32_t* to = a.out_table + static_cast<int64_t>(b) * a.out_table_stride;
    const int reads = (n + kPage - 1) / kPage, writes = min((min(n, a.budget) + kPage - 1) / kPage, a.out_table_pages);
    for (int t = lane; t < writes; t += 32) {
      const int page = to[t];
#pragma unroll 4
      for (int r = warp; r < reads; r += kEvThreads / 32) both |= from[r] == page && page >= 0;
    }
  }
  for (int base = 0; base < a.budget - need; base += kEvThreads) {
    const int i = base + tid;
    const bool there = i < recent;
    if (base > 0) y = there && w_out != nullptr ? w[front + i] : 0.f;
    __syncthreads();
    if (i < a.budget - need) {
      kept[need + i] = there ? front + i : -1;
      if (w_out != nullptr) w_out[need + i] = y;
    }
    __syncthreads();
  }
  int64_t rest = a.budget;
  if (apart && __syncthreads_or(both)) {
    // it keeps nothing, so that no row moves
    for (int i = tid; i < a.budget; i += kEvThreads) kept[i] = -1;
    rest = 0;
    if (tid == 0) report_status(MDB_STATUS_BAD_PAGE);
  }
  // Behind the budget lie no keys: with weights_out the weights, what lay there would be the past of keys that are appended later.  (All of
  // w has been read.)
  if (w_out != nullptr)
    for (int64_t i = rest + tid; i < out_cols; i += kEvThreads) w_out[i] = 0.f;
}

// Byte offset of a place in the pool, or -1.
__device__ __forceinline__ int64_t ev_place(const int32_t* table, int pages, int num_pages, int i, int64_t token_bytes) {
  const int p = i / kPage;
  const int page = p < pages ? table[p] : -1;
  if (page < 0 || page >= num_pages) return -1;
  return (static_cast<int64_t>(page) * kPage + i % kPage) * token_bytes;
}

// `slice` pieces of 16 bytes of rows of one (request, key head) of K or V: of kEvMoveRows of them from kEvMoveRows blockIdx.y on, or
// of all, kEvStepRows at a time.
template <bool IN_PLACE>
__global__ void __launch_bounds__(kEvMoveThreads) evict_move_kernel(const mdb_kv_evict_args a, const int slice) {
  constexpr int kRows = IN_PLACE ? kEvStepRows : kEvMoveRows;
  __shared__ int64_t places[2][kRows];               // old and new byte offset of a row; old -1: stays
  pdl_launch_dependents();
  const int pieces = a.row_bytes / 16, parts = pieces / slice;
  int rest = blockIdx.x;
  const int part = rest % parts; rest /= parts;
  const bool values = rest & 1; rest >>= 1;
  const int pair = rest, b = pair / a.kv_heads, h = pair % a.kv_heads, tid = threadIdx.x;
  unsigned char* cache = static_cast<unsigned char*>(values ? a.v_cache : a.k_cache);
  const int32_t* kept = a.kept + static_cast<int64_t>(pair) * a.budget;
  const int32_t* from = a.block_table + static_cast<int64_t>(b) * a.table_stride;
  const int32_t* to = IN_PLACE ? from : a.out_table + static_cast<int64_t>(b) * a.out_table_stride;
  const int to_pages = a.out_table == nullptr ? a.table_pages : a.out_table_pages;
  const int64_t token_bytes = static_cast<int64_t>(a.kv_heads) * a.row_bytes;
  const int piece = tid % slice, r0 = tid / slice, rows = kEvMoveThreads / slice;
  cache += static_cast<int64_t>(h) * a.row_bytes + (part * slice + piece) * 16;
  pdl_wait();
  if (blockIdx.y == 0 && part == 0 && !values && h == 0 && tid == 0) {
    // (the lengths are read by the kernel in front alone, so that they may be replaced here)
    const int64_t most = min(static_cast<int64_t>(a.table_pages) * kPage, static_cast<int64_t>(a.weight_cols));
    const int stay = max(0, static_cast<int>(min(static_cast<int64_t>(min(a.seqlens[b], a.budget)), most)));
    a.seqlens_out[b] = kept[0] < 0 ? 0 : stay;
  }
  bool bad = false;
  for (int base = IN_PLACE ? 0 : blockIdx.y * kEvMoveRows; base < a.budget; base += kRows) {
    for (int r = tid; r < kRows; r += kEvMoveThreads) {
      const int i = base + r, old = i < a.budget ? kept[i] : -1;
      int64_t src = -1, dst = -1;
      if (old >= 0 && !(IN_PLACE && old == i)) {
        src = ev_place(from, a.table_pages, a.num_pages, old, token_bytes);
        dst = ev_place(to, to_pages, a.num_pages, i, token_bytes);
        if (src < 0 || dst < 0) { bad = true; src = -1; }
      }
      places[0][r] = src;
      places[1][r] = dst;
    }
    __syncthreads();
    for (int r = r0; r < kRows; r += rows * kEvMovePieces) {
      uint4 x[kEvMovePieces];
#pragma unroll
      for (int j = 0; j < kEvMovePieces; ++j) {
        const int i = r + j * rows;
        const int64_t src = i < kRows ? places[0][i] : -1;
        if (src >= 0) x[j] = *reinterpret_cast<const uint4*>(cache + src);
      }
      if (IN_PLACE) __syncthreads();                       // (every thread takes as many turns)
#pragma unroll
      for (int j = 0; j < kEvMovePieces; ++j) {
        const int i = r + j * rows;
        if (i < kRows && places[0][i] >= 0) *reinterpret_cast<uint4*>(cache + places[1][i]) = x[j];
      }
    }
    if (!IN_PLACE) break;
    __syncthreads();
  }
  if (bad) report_status(MDB_STATUS_BAD_PAGE);
}

}  // namespace mdb

using namespace mdb;

extern "C" int mdb_kv_evict(const mdb_kv_evict_args* args, mdb_stream_t stream) {
  MDB_REQUIRE(args != nullptr, MDB_ERR_ARG);
  const mdb_kv_evict_args& a = *args;
  const bool same = a.weights_out == a.weights && a.weight_out_row == a.weight_row && a.weight_out_head == a.weight_head && a.weight_cols > a.budget;
  return mdb_kv_evict_wide(args, same ? a.weight_cols : a.budget, stream);
}

extern "C" int mdb_kv_evict_wide(const mdb_kv_evict_args* args, int64_t weight_out_cols, mdb_stream_t stream) {
  MDB_REQUIRE(args != nullptr, MDB_ERR_ARG);
  const mdb_kv_evict_args a = *args;
  MDB_REQUIRE(a.bs >= 0 && a.kv_heads > 0 && a.row_bytes > 0 && a.budget > 0 && a.recent >= 0 && a.recent <= a.budget && a.num_pages > 0 &&
                  a.table_pages > 0 && (a.table_stride >= a.table_pages || a.bs <= 1) && a.weight_cols > 0,
              MDB_ERR_ARG);
  if (a.bs == 0) return MDB_OK;
  MDB_REQUIRE(a.weights_out == nullptr || weight_out_cols >= a.budget, MDB_ERR_ARG);
  MDB_REQUIRE(a.k_cache && a.v_cache && a.weights && a.seqlens && a.seqlens_out && a.block_table && a.kept, MDB_ERR_ARG);
  MDB_REQUIRE(a.out_table == nullptr || (a.out_table_pages > 0 && (a.out_table_stride >= a.out_table_pages || a.bs <= 1)), MDB_ERR_ARG);
  MDB_REQUIRE(a.row_bytes % 16 == 0 && mdb_aligned16(a.k_cache) && mdb_aligned16(a.v_cache), MDB_ERR_ALIGN);
  MDB_REQUIRE(static_cast<int64_t>(a.bs) * a.kv_heads <= 32767 && a.budget <= (1 << 23) && a.table_pages <= (1 << 22) && a.out_table_pages <= (1 << 22),
              MDB_ERR_UNSUPPORTED);
  // rows of weights that lie on one another
  MDB_REQUIRE(a.weights_out == nullptr || mdb_pieces_apart(a.bs, a.weight_out_row, a.kv_heads, a.weight_out_head, weight_out_cols), MDB_ERR_ARG);
  MDB_REQUIRE(a.row_bytes <= 4096, MDB_ERR_UNSUPPORTED);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int pairs = a.bs * a.kv_heads;
  // the same table once more: in place (a table that starts at the same entry with rows further apart is another one)
  const bool apart = a.out_table != nullptr && (a.out_table != a.block_table || (a.out_table_stride != a.table_stride && a.bs > 1));
  int rc = mdb_launch(evict_select_kernel, dim3(pairs), dim3(kEvThreads), 0, st, a, weight_out_cols, apart);
  if (rc != MDB_OK) return rc;
  // slices of a power of two of pieces that divides the row, as wide as it goes; in place narrower, down to 32 bytes, until the
  // SMs have two CTAs each (one request of 4100 keys, eight heads: 28 us whole rows, 15 us slices; 16 of 8192 alike)
  const int pieces = a.row_bytes / 16;
  int slice = 1;
  while (slice < 32 && pieces % (2 * slice) == 0) slice *= 2;
  if (!apart) {
    while (slice > 2 && static_cast<int64_t>(pairs) * 2 * (pieces / slice) < 2 * at_sm_count()) slice /= 2;
    return mdb_launch(evict_move_kernel<true>, dim3(2 * pairs * (pieces / slice)), dim3(kEvMoveThreads), 0, st, a, slice);
  }
  return mdb_launch(evict_move_kernel<false>, dim3(2 * pairs * (pieces / slice), (a.budget + kEvMoveRows - 1) / kEvMoveRows), dim3(kEvMoveThreads), 0, st, a,
                    slice);
}
