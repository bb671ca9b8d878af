// Rotary positions of queries and keys, with the store of keys and values into the paged cache (no norms; the fused forms of the
// layer stacks are in elementwise.cu and window_attention.cu).
//
// With t = position * inv_freq[i], the channel pair i of a head, (i, i + rot / 2) or (2 i, 2 i + 1), becomes
// scale * (a cos t - b sin t, b cos t + a sin t); `inverse` turns by -t, which is the gradient of the turn.  Channels from
// rot on pass.  Angles are products of 64 bits, taken to a fraction of a turn there: at position 131072 a product of 32 bits is
// off by up to 2^-8 radian.  What is left is a number in [-1, 1] half turns, whose sine and cosine need no reduction.
//
// A CTA takes some tokens: sines and cosines of their pairs once, into shared memory, for all heads.  A thread has one piece of 16 bytes
// (half layout: two) of one head, whose place it works out once, and goes through the tokens with it, loads of kReBatch tokens (half
// layout: of half as many) in front of their stores.  It is bound by memory: 16384 tokens of 40 heads, a quarter of 128 channels turned,
// 56.5 us = 5.9 TB/s (indices worked out for every token: 66); less than a round of CTAs by the trip to positions, sines and rows (32
// tokens: 2.7 us).
#include "mdb_common.cuh"

namespace mdb {

constexpr int kReThreads = 640, kReTokens = 16, kReBatch = 4;         // at most; tokens whose loads are in flight together

template <typename T>
struct ReVec;
template <>
struct ReVec<float> {
  static constexpr int kWide = 4;
  __device__ static void unpack(const uint4& u, float (&x)[4]) {
    x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y); x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
  }
  __device__ static uint4 pack(const float (&x)[4]) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};
template <>
struct ReVec<bf16> {
  static constexpr int kWide = 8;
  __device__ static void unpack(const uint4& u, float (&x)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack_bf16x2(w[i]);
      x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
  }
  __device__ static uint4 pack(const float (&x)[8]) {
    return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
  }
};
__device__ __forceinline__ float re_load(const float* p) { return *p; }
__device__ __forceinline__ float re_load(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void re_store(float* p, float v) { *p = v; }
__device__ __forceinline__ void re_store(bf16* p, float v) { *p = __float2bfloat16_rn(v); }

// Pieces of a head: pairs of vectors (half layout) or vectors that hold whole pairs, then what passes.  WIDE: 16 bytes; otherwise
// single numbers (sizes, strides or addresses that are no multiples of 16 bytes).
template <typename T, bool WIDE, bool PAIRS, int BATCH>
__global__ void __launch_bounds__(kReThreads, 2) rotary_embed_kernel(const mdb_rotary_embed_args a, const int tokens) {
  constexpr int V = WIDE ? ReVec<T>::kWide : 1;
  extern __shared__ float2 re_cs[];                        // [tokens][rot / 2]
  __shared__ int64_t slots[kReTokens];                     // -1: skipped
  const int half = a.rot_dims / 2, tid = threadIdx.x;
  const int tok0 = blockIdx.x * tokens, count = min(tokens, a.n - tok0);
  pdl_launch_dependents();
  // pieces of a head that turn, of one that turns or passes, of one that passes
  const int turned = PAIRS ? (WIDE ? a.rot_dims / V : half) : half / V;
  const int pieces = turned + (a.dim - a.rot_dims) / V, whole = a.dim / V;
  const int turning = (a.heads + a.kv_heads) * pieces, columns = turning + (a.v != nullptr ? a.kv_heads * whole : 0);
  pdl_wait();
  for (int i = tid; i < count * half; i += blockDim.x) {
    const int t = i / half, p = i - t * half;
    const double turns = static_cast<double>(a.positions[tok0 + t]) * (a.inv_freq[p] * 0.15915494309189533577);
    float s, c;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
    re_cs[i] = make_float2(c * a.scale, (a.inverse ? -s : s) * a.scale);
  }
  if (a.slots != nullptr && tid < count) {
    const int64_t slot = a.slots[tok0 + tid];
    const bool there = slot >= 0 && slot < a.num_slots;
    if (!there && slot != -1) report_status(MDB_STATUS_BAD_SLOT);
    slots[tid] = there ? slot : -1;
  }
  __syncthreads();
  for (int column = tid; column < columns; column += blockDim.x) {
    const bool value = column >= turning;
    const int per = value ? whole : pieces, at = value ? column - turning : column;
    int h = at / per, u = at - h * per;
    const bool turn = !value && u < turned, query = !value && h < a.heads;
    if (!value && !query) h -= a.heads;
    // offset of the piece's first vector in a head
    const int c = value ? u * V : turn ? (PAIRS && !WIDE ? 2 * u : u * V) : a.rot_dims + (u - turned) * V;
    const int64_t from = query ? a.q_row : value ? a.v_row : a.k_row;
    const T* src = static_cast<const T*>(query ? a.q : value ? a.v : a.k) + tok0 * from + h * (query ? a.q_head : value ? a.v_head : a.k_head) + c;
    const bool stored = !query && a.slots != nullptr;
    const int64_t to = stored ? static_cast<int64_t>(a.kv_heads) * a.dim : query ? a.q_out_row : a.k_out_row;
    T* dst = static_cast<T*>(stored ? (value ? a.v_cache : a.k_cache) : query ? a.q_out : a.k_out) +
             (stored ? h * a.dim : tok0 * to + h * (query ? a.q_out_head : a.k_out_head)) + c;
    const float2* cs = re_cs + (PAIRS && WIDE ? u * V / 2 : u * V);
    if (WIDE) {
      for (int t0 = 0; t0 < count; t0 += BATCH) {
        uint4 x[BATCH], y[PAIRS ? 1 : BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          if (t0 + j >= count) break;
          x[j] = *reinterpret_cast<const uint4*>(src + (t0 + j) * from);
          if (!PAIRS && turn) y[j] = *reinterpret_cast<const uint4*>(src + (t0 + j) * from + half);
        }
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          if (t0 + j >= count) break;
          const int64_t row = stored ? slots[t0 + j] : t0 + j;
          if (row < 0) continue;
          constexpr int W = ReVec<T>::kWide;
          T* const d = dst + row * to;
          const float2* const f = cs + (t0 + j) * half;
          if (turn) {
            float v[W];
            ReVec<T>::unpack(x[j], v);
            if (PAIRS) {
#pragma unroll
              for (int i = 0; i < W; i += 2) {
                const float2 g = f[i / 2];
                const float lo = v[i], hi = v[i + 1];
                v[i] = lo * g.x - hi * g.y;
                v[i + 1] = hi * g.x + lo * g.y;
              }
            } else {
              float z[W];
              ReVec<T>::unpack(y[PAIRS ? 0 : j], z);
#pragma unroll
              for (int i = 0; i < W; ++i) {
                const float2 g = f[i];
                const float lo = v[i], hi = z[i];
                v[i] = lo * g.x - hi * g.y;
                z[i] = hi * g.x + lo * g.y;
              }
              *reinterpret_cast<uint4*>(d + half) = ReVec<T>::pack(z);
            }
            x[j] = ReVec<T>::pack(v);
          }
          *reinterpret_cast<uint4*>(d) = x[j];
        }
      }
    } else {
      for (int t = 0; t < count; ++t) {
        const int64_t row = stored ? slots[t] : t;
        if (row < 0) continue;
        const T* const x = src + t * from;
        T* const d = dst + row * to;
        if (turn) {
          const int other = PAIRS ? 1 : half;
          const float2 g = cs[t * half];
          const float lo = re_load(x), hi = re_load(x + other);
          re_store(d, lo * g.x - hi * g.y);
          re_store(d + other, hi * g.x + lo * g.y);
        } else {
          d[0] = x[0];
        }
      }
    }
  }
}

template <typename T>
static int re_launch(const mdb_rotary_embed_args& a, cudaStream_t st) {
  constexpr int W = ReVec<T>::kWide;
  const auto even = [&](const void* p, int64_t row, int64_t head) { return p == nullptr || (mdb_aligned16(p) && row % W == 0 && head % W == 0); };
  const bool wide = a.dim % W == 0 && (a.interleaved ? a.rot_dims : a.rot_dims / 2) % W == 0 && even(a.q, a.q_row, a.q_head) &&
                    even(a.k, a.k_row, a.k_head) && even(a.v, a.v_row, a.v_head) && even(a.q_out, a.q_out_row, a.q_out_head) &&
                    even(a.k_out, a.k_out_row, a.k_out_head) && even(a.k_cache, 0, 0) && even(a.v_cache, 0, 0);
  const int v = wide ? W : 1;
  const int pieces = (a.interleaved && wide ? a.rot_dims / v : a.rot_dims / 2 / v) + (a.dim - a.rot_dims) / v;
  const int columns = (a.heads + a.kv_heads) * pieces + (a.v != nullptr ? a.kv_heads * (a.dim / v) : 0);
  // turns of about as many columns each, whole warps
  const int turns = (columns + kReThreads - 1) / kReThreads, threads = ((columns + turns - 1) / turns + 31) / 32 * 32;
  // a token per CTA while all CTAs are resident at once (48 registers a thread), then as few full rounds as there can be
  const int64_t resident = at_sm_count() * static_cast<int64_t>(65536 / (48 * threads)), rounds = (a.n + resident * kReTokens - 1) / (resident * kReTokens);
  int tokens = static_cast<int>((a.n + resident * rounds - 1) / (resident * rounds));
  while (tokens > 1 && sizeof(float2) * tokens * (a.rot_dims / 2) > 40 * 1024) tokens /= 2;
  const dim3 grid((a.n + tokens - 1) / tokens), block(threads);
  const size_t smem = sizeof(float2) * tokens * (a.rot_dims / 2);
  const auto go = [&](auto kernel) { return mdb_launch(kernel, grid, block, smem, st, a, tokens); };
  if (!wide) return a.interleaved ? go(rotary_embed_kernel<T, false, true, 1>) : go(rotary_embed_kernel<T, false, false, 1>);
  if (tokens == 1) return a.interleaved ? go(rotary_embed_kernel<T, true, true, 1>) : go(rotary_embed_kernel<T, true, false, 1>);
  return a.interleaved ? go(rotary_embed_kernel<T, true, true, kReBatch>) : go(rotary_embed_kernel<T, true, false, kReBatch / 2>);
}

}  // namespace mdb

using namespace mdb;

extern "C" int mdb_rotary_embed(const mdb_rotary_embed_args* args, mdb_stream_t stream) {
  MDB_REQUIRE(args != nullptr, MDB_ERR_ARG);
  const mdb_rotary_embed_args a = *args;
  MDB_REQUIRE(a.n >= 0 && a.heads > 0 && a.kv_heads >= 0 && a.dim > 0 && a.rot_dims >= 0 && a.rot_dims <= a.dim && a.rot_dims % 2 == 0,
              MDB_ERR_ARG);
  MDB_REQUIRE(a.dtype == MDB_BF16 || a.dtype == MDB_F32, MDB_ERR_ARG);
  if (a.n == 0) return MDB_OK;
  MDB_REQUIRE(a.q && a.q_out && a.positions && (a.rot_dims == 0 || a.inv_freq), MDB_ERR_ARG);
  if (a.slots != nullptr) MDB_REQUIRE(a.kv_heads > 0 && a.k && a.k_cache && (!a.v || a.v_cache) && a.num_slots > 0, MDB_ERR_ARG);
  else MDB_REQUIRE((a.kv_heads == 0 || (a.k && a.k_out)) && a.v == nullptr, MDB_ERR_ARG);
  MDB_REQUIRE(a.dim <= 1024 && a.heads <= 65536 && a.kv_heads <= 65536, MDB_ERR_UNSUPPORTED);
  // heads of an output that lie on one another
  MDB_REQUIRE(mdb_pieces_apart(a.n, a.q_out_row, a.heads, a.q_out_head, a.dim), MDB_ERR_ARG);
  if (a.slots == nullptr && a.kv_heads > 0) MDB_REQUIRE(mdb_pieces_apart(a.n, a.k_out_row, a.kv_heads, a.k_out_head, a.dim), MDB_ERR_ARG);
  MDB_REQUIRE(static_cast<int64_t>(a.heads) + 2 * static_cast<int64_t>(a.kv_heads) <= 65536, MDB_ERR_UNSUPPORTED);
  return a.dtype == MDB_BF16 ? re_launch<bf16>(a, static_cast<cudaStream_t>(stream)) : re_launch<float>(a, static_cast<cudaStream_t>(stream));
}
