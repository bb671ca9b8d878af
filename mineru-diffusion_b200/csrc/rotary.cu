// Rotary positions of queries and keys, with the store of keys and values into the paged cache (no norms; the fused forms of the
// layer stacks are in elementwise.cu and window_attention.cu).
//
// With t = position * inv_freq[i], the channel pair i of a head, (i, i + rot / 2) or (2 i, 2 i + 1), becomes
// scale * (a cos t - b sin t, b cos t + a sin t); `inverse` turns by -t, which is the gradient of the turn.  Channels from
// rot on pass.  Angles are products of 64 bits, taken to a fraction of a turn there: at position 131072 a product of 32 bits is
// off by up to 2^-8 radian.  What is left is a number in [-1, 1] half turns, whose sine and cosine need no reduction.
//
// A CTA takes `tokens` tokens: sines and cosines of their pairs once, into shared memory, for all heads.  Threads lie in rows of
// `width` (a power of two) along a head's pieces of 16 bytes, so that no index needs a division but a row's token.
// It is bound by memory.  Measured: see the table of the cases; one token per CTA below 2 x 148 x 8 of them, four from there on.
#include "mdb_common.cuh"

namespace mdb {

constexpr int kReThreads = 256;
constexpr int kReManyTokens = 4;

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
template <typename T, bool WIDE, bool PAIRS>
__global__ void __launch_bounds__(kReThreads) rotary_embed_kernel(const mdb_rotary_embed_args a, const int tokens, const int width) {
  constexpr int V = WIDE ? ReVec<T>::kWide : 1;
  extern __shared__ float2 re_cs[];                        // [tokens][rot / 2]
  const int half = a.rot_dims / 2, tid = threadIdx.x;
  const int tok0 = blockIdx.x * tokens, count = min(tokens, a.n - tok0);
  pdl_launch_dependents();
  pdl_wait();
  for (int i = tid; i < count * half; i += kReThreads) {
    const int t = i / half, p = i - t * half;
    const double turns = static_cast<double>(a.positions[tok0 + t]) * (a.inv_freq[p] * 0.15915494309189533577);
    float s, c;
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
    re_cs[i] = make_float2(c * a.scale, (a.inverse ? -s : s) * a.scale);
  }
  __syncthreads();

  // pieces of a head that turn, and of one that turns or passes
  const int turned = PAIRS ? (WIDE ? a.rot_dims / V : half) : half / V;
  const int pieces = turned + (a.dim - a.rot_dims) / V;
  const int heads = a.heads + a.kv_heads + (a.v != nullptr ? a.kv_heads : 0);
  const float per_head = 1.0f / static_cast<float>(heads);
  const int rows = kReThreads / width, u0 = tid & (width - 1);
  for (int r = tid / width; r < count * heads; r += rows) {
    const int t = static_cast<int>((static_cast<float>(r) + 0.5f) * per_head), head = r - t * heads;   // exact: r < 2^14
    const int64_t row = tok0 + t;
    const T* src;
    T* dst;
    int h = head;
    bool turn = true;
    if (head < a.heads) {
      src = static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head;
      dst = static_cast<T*>(a.q_out) + row * a.q_out_row + h * a.q_out_head;
    } else {
      h = head - a.heads;
      turn = h < a.kv_heads;
      if (!turn) h -= a.kv_heads;
      src = turn ? static_cast<const T*>(a.k) + row * a.k_row + h * a.k_head : static_cast<const T*>(a.v) + row * a.v_row + h * a.v_head;
      if (a.slots != nullptr) {
        const int64_t slot = a.slots[row];
        if (slot < 0 || slot >= a.num_slots) {
          if (slot != -1 && u0 == 0) report_status(MDB_STATUS_BAD_SLOT);
          continue;
        }
        dst = static_cast<T*>(turn ? a.k_cache : a.v_cache) + (slot * a.kv_heads + h) * a.dim;
      } else {
        dst = static_cast<T*>(a.k_out) + row * a.k_out_row + h * a.k_out_head;
      }
    }
    const float2* cs = re_cs + t * half;
    const int end = turn ? pieces : a.dim / V;
    for (int u = u0; u < end; u += width) {
      if (!turn || u >= turned) {
        const int c = turn ? a.rot_dims + (u - turned) * V : u * V;
        if (WIDE) *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(src + c);
        else dst[c] = src[c];
      } else if (WIDE && PAIRS) {
        constexpr int W = ReVec<T>::kWide;
        float x[W];
        ReVec<T>::unpack(*reinterpret_cast<const uint4*>(src + u * V), x);
#pragma unroll
        for (int i = 0; i < W; i += 2) {
          const float2 f = cs[(u * V + i) / 2];
          const float lo = x[i], hi = x[i + 1];
          x[i] = lo * f.x - hi * f.y;
          x[i + 1] = hi * f.x + lo * f.y;
        }
        *reinterpret_cast<uint4*>(dst + u * V) = ReVec<T>::pack(x);
      } else if (WIDE) {
        constexpr int W = ReVec<T>::kWide;
        float x[W], y[W];
        ReVec<T>::unpack(*reinterpret_cast<const uint4*>(src + u * V), x);
        ReVec<T>::unpack(*reinterpret_cast<const uint4*>(src + half + u * V), y);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float2 f = cs[u * V + i];
          const float lo = x[i], hi = y[i];
          x[i] = lo * f.x - hi * f.y;
          y[i] = hi * f.x + lo * f.y;
        }
        *reinterpret_cast<uint4*>(dst + u * V) = ReVec<T>::pack(x);
        *reinterpret_cast<uint4*>(dst + half + u * V) = ReVec<T>::pack(y);
      } else {
        const int c0 = PAIRS ? 2 * u : u, c1 = PAIRS ? 2 * u + 1 : u + half;
        const float2 f = cs[u];
        const float lo = re_load(src + c0), hi = re_load(src + c1);
        re_store(dst + c0, lo * f.x - hi * f.y);
        re_store(dst + c1, hi * f.x + lo * f.y);
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
  int width = 1;
  while (width < pieces && width < kReThreads) width *= 2;
  const int tokens = a.n >= 2 * 148 * 8 ? kReManyTokens : 1;
  const dim3 grid((a.n + tokens - 1) / tokens), block(kReThreads);
  const size_t smem = sizeof(float2) * tokens * (a.rot_dims / 2);
  if (wide)
    return a.interleaved ? mdb_launch(rotary_embed_kernel<T, true, true>, grid, block, smem, st, a, tokens, width)
                         : mdb_launch(rotary_embed_kernel<T, true, false>, grid, block, smem, st, a, tokens, width);
  return a.interleaved ? mdb_launch(rotary_embed_kernel<T, false, true>, grid, block, smem, st, a, tokens, width)
                       : mdb_launch(rotary_embed_kernel<T, false, false>, grid, block, smem, st, a, tokens, width);
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
  // a row's index has to be exact in the kernel's fp32 division, and the sines of four tokens to fit 48 KB
  MDB_REQUIRE(a.dim <= 1024 && static_cast<int64_t>(a.heads) + 2 * static_cast<int64_t>(a.kv_heads) <= 2048, MDB_ERR_UNSUPPORTED);
  return a.dtype == MDB_BF16 ? re_launch<bf16>(a, static_cast<cudaStream_t>(stream)) : re_launch<float>(a, static_cast<cudaStream_t>(stream));
}
