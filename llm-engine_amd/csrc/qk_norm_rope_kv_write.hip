// Per-head RMSNorm of q and k, RoPE and the K/V cache-write scatter in one
// launch, from the stacked QKV projection rows:
//     x = row (+ bias);  y = x / sqrt(mean_j x_j^2 + eps) * w  over each q and
//     k head (w of q or of k);  a' = a cos - b sin, b' = b cos + a sin with
//     a = y_i, b = y_{i + half};  v = x
// all in fp32, each stored value rounded once.
//
// A head is held by head_dim / (2 W) adjacent lanes: a lane has W elements of
// its lower half and the W that they rotate with (W = 8: two 16-byte pieces
// of a 16-bit row), so the mean is one reduction inside the wave, and neither
// the norm nor the rotation goes through memory. A lane's dims are the same for
// all its heads, so its cos and sin stay in registers.
//
// Bound by the bytes of the rows. A workgroup takes a token, all heads; while
// all workgroups run at once anyway, several share a token, a head per lane
// group, so that no second head waits for the first one's trip to memory (32 +
// 2 x 8 heads of 128, 15 fp32 rows: 3.2 us, unshared 4.1; 905 fp16 rows 8.1,
// 8.6). Past that the copies of cos and sin cost more (1371 fp32 rows: 14.3 us,
// 15.1 shared). 4096 bf16 rows of that shape take 24.5 us, 4.2 TB/s, where a
// copy of 1 GiB reaches 5.0; 3898 rows of 10 + 2 x 10 heads 4.99 TB/s.
#include "le_common.h"
#include "le_internal.h"

namespace le {
namespace {

constexpr int kNormThreads = 256;
constexpr int kResident = 2048;  // workgroups that run at once: 256 CUs of 32 waves

template <typename T, int W> __device__ __forceinline__ void load_w(const T* p, float* o) {
  if constexpr (W == 8) elem<T>::load8(p, o);
  else elem<T>::load4(p, o);
}
template <typename T, int W> __device__ __forceinline__ void store_w(T* p, const float* v) {
  if constexpr (W == 8) elem<T>::store8(p, v);
  else elem<T>::store4(p, v);
}

// LANES > 0: lanes of a head, known (head_dim = 2 W LANES). 0: `lanes`, a
// power of two of at least head_dim / (2 W); lanes past the head hold nothing.
template <typename T, typename C, int W, int LANES>
__global__ __launch_bounds__(kNormThreads) void qk_norm_rope_kernel(QkNormParams p) {
  const int lanes = LANES > 0 ? LANES : p.lanes;
  const int t = blockIdx.x;
  const int hd = LANES > 0 ? 2 * W * LANES : p.head_dim, half = hd >> 1;
  const int unit0 = (blockIdx.y * kNormThreads + threadIdx.x) / lanes, per_step = gridDim.y * kNormThreads / lanes;
  const int i = (threadIdx.x & (lanes - 1)) * W;  // this lane's dims: [i, i + W) and the same past half
  const bool live = LANES > 0 || i < half;
  const int at = live ? i : 0;
  const int pos = p.positions[t];
  const int64_t slot = p.slots[t];
  const bool pos_ok = pos >= 0 && pos < p.max_pos;
  const bool kv_ok = pos_ok && slot >= 0 && slot < p.num_slots;
  const int nh = p.q_heads, nkv = p.kv_heads;
  const T* row = static_cast<const T*>(p.qkv) + static_cast<int64_t>(t) * p.row_stride;
  const int64_t tab = static_cast<int64_t>(pos_ok ? pos : 0) * half + at;
  float c[W], s[W];
  load_w<float, W>(p.cos_t + tab, c);
  load_w<float, W>(p.sin_t + tab, s);
  // heads: q, then k, then v (copied)
  for (int u = unit0; u < nh + 2 * nkv; u += per_step) {
    const int off = u * hd + at;
    float a[W], b[W];
    load_w<T, W>(row + off, a);
    load_w<T, W>(row + off + half, b);
    if (p.bias) {
#pragma unroll
      for (int e = 0; e < W; e++) {
        a[e] += p.bias[off + e];
        b[e] += p.bias[off + half + e];
      }
    }
    if (u < nh + nkv) {
      float ss = 0.f;
      if (live) {
#pragma unroll
        for (int e = 0; e < W; e++) ss += a[e] * a[e] + b[e] * b[e];
      }
      if constexpr (LANES > 0) {
        ss = group_sum<LANES>(ss);
      } else {
        for (int d = 1; d < lanes; d <<= 1) ss += __shfl_xor(ss, d, kWave);
      }
      const float r = 1.0f / sqrtf(ss / hd + p.eps);
      const float* w = (u < nh ? p.q_norm : p.k_norm) + at;
      float wa[W], wb[W];
      load_w<float, W>(w, wa);
      load_w<float, W>(w + half, wb);
#pragma unroll
      for (int e = 0; e < W; e++) {
        const float x = a[e] * r * wa[e], y = b[e] * r * wb[e];
        a[e] = pos_ok ? x * c[e] - y * s[e] : 0.f;
        b[e] = pos_ok ? y * c[e] + x * s[e] : 0.f;
      }
    }
    if (!live) continue;
    if (u < nh) {
      T* dst = static_cast<T*>(p.q_out) + static_cast<int64_t>(t) * nh * hd + off;
      store_w<T, W>(dst, a);
      store_w<T, W>(dst + half, b);
    } else if (kv_ok) {
      const int h = u - nh;
      C* cache = static_cast<C*>(h < nkv ? p.k_cache : p.v_cache);
      C* dst = cache + (slot * nkv + (h < nkv ? h : h - nkv)) * hd + at;
      store_w<C, W>(dst, a);
      store_w<C, W>(dst + half, b);
    }
  }
}

}  // namespace

hipError_t qk_norm_rope_kv_write(const QkNormParams& in, int act_dtype, int cache_dtype, hipStream_t stream) {
  QkNormParams p = in;
  const auto grid = [&](int lanes) {
    const int64_t split = (static_cast<int64_t>(p.q_heads + 2 * p.kv_heads) * lanes + kNormThreads - 1) / kNormThreads;
    return dim3(static_cast<unsigned>(p.n_tokens), p.n_tokens * split <= kResident ? static_cast<unsigned>(split) : 1u);
  };
  return with_dtype(act_dtype, [&](auto a) {
    return with_dtype(cache_dtype, [&](auto c) {
      using T = decltype(a);
      using C = decltype(c);
      if (p.head_dim == 64) {
        qk_norm_rope_kernel<T, C, 8, 4><<<grid(4), kNormThreads, 0, stream>>>(p);
      } else if (p.head_dim == 128) {
        qk_norm_rope_kernel<T, C, 8, 8><<<grid(8), kNormThreads, 0, stream>>>(p);
      } else {
        p.lanes = 1;
        while (p.lanes * 8 < p.head_dim) p.lanes *= 2;
        qk_norm_rope_kernel<T, C, 4, 0><<<grid(p.lanes), kNormThreads, 0, stream>>>(p);
      }
      return hipGetLastError();
    });
  });
}

}  // namespace le
