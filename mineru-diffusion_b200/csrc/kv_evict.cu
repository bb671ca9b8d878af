// Eviction from the paged cache by the weight its keys have received (key_weights.cu).
//
// Per request and key head: of n keys the last `recent` stay, and of those in front the budget - recent with the largest weight
// (NaN counts as the lowest, the lowest index wins a tie).  The rows that stay are packed, in order, into the first places of the
// request's pages, or of other pages; their weights move with them.
//
//   evict_select_kernel   a CTA per (request, key head).  Radix selection over the weights' bits in order (11, 11 and 10 bits, counts in
//                         shared memory): after it the key of the last one that stays is known, and how many of its equals do.
//                         Then one walk in order: 8 neighbouring weights per thread, sums over the CTA, places written.
//   evict_move_kernel     rows of K and V.  To other pages: any order, chunks of rows per CTA.  In place a row's new place is never
//                         behind its old one, so a CTA that has a slice of the channels of all rows walks them in order, loads
//                         of a step in front of its stores.
//
// Bound by memory (rows read and written once); the selection reads the weights from L1 after its first pass.
#include "mdb_common.cuh"

namespace mdb {

constexpr int kEvThreads = 1024, kEvPerThread = 8, kEvTile = kEvThreads * kEvPerThread;
constexpr int kEvBins = 2048;
constexpr int kEvMoveThreads = 256, kEvMoveRows = 8;       // pieces of 16 bytes in flight per thread

// Bits that order like the numbers: negative ones upside down, -0 as 0, NaN lowest.
__device__ __forceinline__ uint32_t ev_key(float w) {
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive sums over the CTA of two counts per thread, packed as 16 bits each (at most kEvTile each).
__device__ __forceinline__ uint32_t ev_sums(uint32_t mine, uint32_t* warp_sums, uint32_t& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += up;
  }
  if (lane == 31) warp_sums[warp] = upto;
  __syncthreads();
  uint32_t w = warp_sums[lane], wu = w;                    // 32 warps
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(0xffffffffu, wu, o);
    if (lane >= o) wu += up;
  }
  all = __shfl_sync(0xffffffffu, wu, 31);
  const uint32_t before = __shfl_sync(0xffffffffu, wu - w, warp);
  __syncthreads();
  return before + upto - mine;
}

__global__ void __launch_bounds__(kEvThreads) evict_select_kernel(const mdb_kv_evict_args a) {
  __shared__ uint32_t counts[kEvBins];
  __shared__ uint32_t warp_sums[32];
  __shared__ uint32_t found[2];
  const int b = blockIdx.x / a.kv_heads, h = blockIdx.x % a.kv_heads, tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  int n = a.seqlens[b];
  const int64_t most = min(static_cast<int64_t>(a.table_pages) * kPage, static_cast<int64_t>(a.weight_cols));
  if (n > most) {
    n = static_cast<int>(most);
    if (tid == 0) report_status(MDB_STATUS_BAD_PAGE);
  }
  n = max(n, 0);
  const float* w = a.weights + b * a.weight_row + h * a.weight_head;
  int32_t* kept = a.kept + (static_cast<int64_t>(b) * a.kv_heads + h) * a.budget;
  float* w_out = a.weights_out == nullptr ? nullptr : a.weights_out + b * a.weight_out_row + h * a.weight_out_head;
  const int stay = min(n, a.budget), recent = min(a.recent, stay);
  const int front = n > a.budget ? n - recent : stay - recent;          // keys that are chosen from, and how many of them
  const int need = stay - recent;
  uint32_t last = 0, equals = 0;                           // key of the last one that stays; how many of its equals stay
  if (need < front && need > 0) {
    uint32_t prefix = 0, left = need;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
      const uint32_t above = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u;
      for (int i = tid; i < bins; i += kEvThreads) counts[i] = 0;
      __syncthreads();
      for (int i = tid; i < front; i += kEvThreads) {
        const uint32_t k = ev_key(w[i]);
        if ((k & above) == prefix) atomicAdd(&counts[(k >> shift) & (bins - 1)], 1u);
      }
      __syncthreads();
      // the bin, from the highest on, in which the left-th key lies: two bins per thread, highest first
      const int hi = bins - 1 - 2 * tid;
      const uint32_t c0 = hi >= 0 ? counts[hi] : 0u, c1 = hi >= 0 ? counts[hi - 1] : 0u;
      uint32_t upto = c0 + c1;
      const int lane = tid & 31, warp = tid >> 5;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
      if (lane == 31) warp_sums[warp] = upto;
      __syncthreads();
      uint32_t base = 0;
      for (int i = 0; i < warp; ++i) base += warp_sums[i];
      upto += base;
      const uint32_t in_front = upto - c0 - c1;
      if (in_front < left && left <= upto) {
        const bool second = left > in_front + c0;
        found[0] = static_cast<uint32_t>(second ? hi - 1 : hi);
        found[1] = left - in_front - (second ? c0 : 0u);
      }
      __syncthreads();
      prefix |= found[0] << shift;
      left = found[1];
      __syncthreads();
    }
    last = prefix;
    equals = left;
  }
  const bool all_stay = need == front;
  // places in order; what a tile reads lies behind all that is written before it (weights_out may be weights)
  uint32_t done = 0, done_equals = 0;
  for (int base = 0; base < front && need > 0; base += kEvTile) {
    float x[kEvPerThread];
    uint32_t above = 0, same = 0, n_above = 0, n_same = 0;
    const int i0 = base + tid * kEvPerThread;
#pragma unroll
    for (int i = 0; i < kEvPerThread; ++i) {
      x[i] = i0 + i < front ? w[i0 + i] : 0.f;
      const uint32_t k = ev_key(x[i]);
      const bool there = i0 + i < front;
      if (there && (all_stay || k > last)) { above |= 1u << i; ++n_above; }
      else if (there && k == last) { same |= 1u << i; ++n_same; }
    }
    uint32_t all;
    const uint32_t before = ev_sums(n_above | n_same << 16, warp_sums, all);
    uint32_t ties = done_equals + (before >> 16);
    uint32_t at = done + (before & 0xffffu) + min(ties, equals);
#pragma unroll
    for (int i = 0; i < kEvPerThread; ++i) {
      const bool tie = same >> i & 1;
      if ((above >> i & 1) || (tie && ties < equals)) {
        kept[at] = i0 + i;
        if (w_out != nullptr) w_out[at] = x[i];
        ++at;
      }
      ties += tie;
    }
    done += all & 0xffffu;
    done_equals += all >> 16;
    __syncthreads();
  }
  for (int base = 0; base < a.budget - need; base += kEvThreads) {
    const int i = base + tid;
    const bool there = i < recent;
    const float x = there && w_out != nullptr ? w[n - recent + i] : 0.f;
    __syncthreads();
    if (i < a.budget - need) {
      kept[need + i] = there ? n - recent + i : -1;
      if (w_out != nullptr) w_out[need + i] = x;
    }
    __syncthreads();
  }
}

// Byte offset of a place in the pool, or -1.
__device__ __forceinline__ int64_t ev_place(const int32_t* table, int pages, int num_pages, int i, int64_t token_bytes) {
  const int p = i / kPage;
  const int page = p < pages ? table[p] : -1;
  if (page < 0 || page >= num_pages) return -1;
  return (static_cast<int64_t>(page) * kPage + i % kPage) * token_bytes;
}

// A CTA: `slice` pieces of 16 bytes of every row in [first, first + rows) of one (request, key head) of K or V.
template <bool IN_PLACE>
__global__ void __launch_bounds__(kEvMoveThreads) evict_move_kernel(const mdb_kv_evict_args a, const int slice, const int rows_per_cta) {
  pdl_launch_dependents();
  pdl_wait();
  const int pair = blockIdx.y >> 1, b = pair / a.kv_heads, h = pair % a.kv_heads, tid = threadIdx.x;
  if (blockIdx.x == 0 && blockIdx.y == 2 * b * a.kv_heads && tid == 0) {
    // (the lengths are read by the kernel in front alone, so that they may be replaced here)
    const int64_t most = min(static_cast<int64_t>(a.table_pages) * kPage, static_cast<int64_t>(a.weight_cols));
    a.seqlens_out[b] = max(0, static_cast<int>(min(static_cast<int64_t>(min(a.seqlens[b], a.budget)), most)));
  }
  unsigned char* cache = static_cast<unsigned char*>(blockIdx.y & 1 ? a.v_cache : a.k_cache);
  const int32_t* kept = a.kept + static_cast<int64_t>(pair) * a.budget;
  const int32_t* from = a.block_table + static_cast<int64_t>(b) * a.table_stride;
  const int32_t* to = IN_PLACE ? from : a.out_table + static_cast<int64_t>(b) * a.out_table_stride;
  const int to_pages = IN_PLACE ? a.table_pages : a.out_table_pages;
  const int64_t token_bytes = static_cast<int64_t>(a.kv_heads) * a.row_bytes;
  const int piece = tid % slice, r0 = tid / slice, rows = kEvMoveThreads / slice;
  const int64_t column = static_cast<int64_t>(h) * a.row_bytes + ((IN_PLACE ? blockIdx.x * slice : 0) + piece) * 16;
  const int first = IN_PLACE ? 0 : blockIdx.x * rows_per_cta, end = IN_PLACE ? a.budget : min(a.budget, first + rows_per_cta);
  bool bad = false;
  const int pieces = a.row_bytes / 16;
  // (to other pages a slice is a whole row, taken in several steps where it has more pieces than the CTA has threads)
  for (int base = first; base < end; base += rows * kEvMoveRows) {
    uint4 x[kEvMoveRows];
    int64_t dst[kEvMoveRows];
#pragma unroll
    for (int j = 0; j < kEvMoveRows; ++j) {
      const int i = base + j * rows + r0;
      const int old = i < end ? kept[i] : -1;
      dst[j] = -1;
      if (old >= 0 && !(IN_PLACE && old == i)) {
        const int64_t src = ev_place(from, a.table_pages, a.num_pages, old, token_bytes);
        const int64_t d = ev_place(to, to_pages, a.num_pages, i, token_bytes);
        if (src >= 0 && d >= 0) {
          dst[j] = d;
          x[j] = *reinterpret_cast<const uint4*>(cache + src + column);
          if (!IN_PLACE)
            for (int p = piece + slice; p < pieces; p += slice)
              *reinterpret_cast<uint4*>(cache + d + column + (p - piece) * 16) =
                  *reinterpret_cast<const uint4*>(cache + src + column + (p - piece) * 16);
        } else {
          bad = true;
        }
      }
    }
    if (IN_PLACE) __syncthreads();
#pragma unroll
    for (int j = 0; j < kEvMoveRows; ++j)
      if (dst[j] >= 0) *reinterpret_cast<uint4*>(cache + dst[j] + column) = x[j];
  }
  if (bad) report_status(MDB_STATUS_BAD_PAGE);
}

}  // namespace mdb

using namespace mdb;

extern "C" int mdb_kv_evict(const mdb_kv_evict_args* args, mdb_stream_t stream) {
  MDB_REQUIRE(args != nullptr, MDB_ERR_ARG);
  const mdb_kv_evict_args a = *args;
  MDB_REQUIRE(a.bs >= 0 && a.kv_heads > 0 && a.row_bytes > 0 && a.budget > 0 && a.recent >= 0 && a.recent <= a.budget && a.num_pages > 0 &&
                  a.table_pages > 0 && (a.table_stride >= a.table_pages || a.bs <= 1) && a.weight_cols > 0,
              MDB_ERR_ARG);
  if (a.bs == 0) return MDB_OK;
  MDB_REQUIRE(a.k_cache && a.v_cache && a.weights && a.seqlens && a.seqlens_out && a.block_table && a.kept, MDB_ERR_ARG);
  MDB_REQUIRE(a.out_table == nullptr || (a.out_table_pages > 0 && (a.out_table_stride >= a.out_table_pages || a.bs <= 1)), MDB_ERR_ARG);
  MDB_REQUIRE(a.row_bytes % 16 == 0 && mdb_aligned16(a.k_cache) && mdb_aligned16(a.v_cache), MDB_ERR_ALIGN);
  MDB_REQUIRE(static_cast<int64_t>(a.bs) * a.kv_heads <= 32767 && a.row_bytes <= 4096 && a.budget <= (1 << 29) && a.table_pages <= (1 << 22) && a.out_table_pages <= (1 << 22),
              MDB_ERR_UNSUPPORTED);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int pairs = a.bs * a.kv_heads;
  int rc = mdb_launch(evict_select_kernel, dim3(pairs), dim3(kEvThreads), 0, st, a);
  if (rc != MDB_OK) return rc;
  const int pieces = a.row_bytes / 16;
  if (a.out_table == nullptr) {
    // slices of at least 32 bytes, a power of two of pieces that divides the row, until the SMs have two CTAs each
    int slice = 1;
    while (slice < 32 && pieces % (2 * slice) == 0) slice *= 2;
    while (slice > 2 && static_cast<int64_t>(pairs) * 2 * (pieces / slice) < 2 * 148) slice /= 2;
    return mdb_launch(evict_move_kernel<true>, dim3(pieces / slice, 2 * pairs), dim3(kEvMoveThreads), 0, st, a, slice, a.budget);
  }
  int slice = 1;                                           // the largest power of two of pieces in a row, up to a warp's worth
  while (slice < 32 && 2 * slice <= pieces) slice *= 2;
  const int rows = kEvMoveThreads / slice * kEvMoveRows;
  return mdb_launch(evict_move_kernel<false>, dim3((a.budget + rows - 1) / rows, 2 * pairs), dim3(kEvMoveThreads), 0, st, a, slice, rows);
}
