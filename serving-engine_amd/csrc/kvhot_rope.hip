// Norms of queries and keys of each head, and their rotation by position.
//
// y = w x / sqrt(mean(x^2) + eps) over a head's D elements, then the first
// `rotary` of them turned pair by pair: (a, b) -> (a cos - b sin, b cos + a sin),
// pairs (i, i + rotary / 2), or (2 i, 2 i + 1) where interleaved, by the
// position's row of a table of cosines and sines.  All of it in fp32 from one
// read of x, rounded once.  Bound by memory: 4 bytes an element in 16 bits.
#include "kvhot_internal.h"

#include <cmath>

namespace kvhot {

struct RopeArgs {
  const void *q, *k;
  void *q_out, *k_out;
  int64_t q_st, q_sh, k_st, k_sh, qo_st, qo_sh, ko_st, ko_sh;
  const void *q_weight, *k_weight;
  const float* table;
  const void* positions;
  int64_t tokens, table_rows;
  int32_t hq, hkv, d, rotary, interleaved, weight_f32, pos_is_int64, vec;
  float eps;
};

// Four values at p.
template <class T>
__device__ inline f32x4 load4(const typename T::storage* p, bool vec) {
  if constexpr (sizeof(typename T::storage) == 4) {
    if (vec) return *reinterpret_cast<const f32x4*>(p);
    return f32x4{p[0], p[1], p[2], p[3]};
  } else {
    u32x2 w;
    if (vec)
      w = *reinterpret_cast<const u32x2*>(p);
    else
      w = u32x2{static_cast<uint32_t>(p[0]) | static_cast<uint32_t>(p[1]) << 16,
                static_cast<uint32_t>(p[2]) | static_cast<uint32_t>(p[3]) << 16};
    return f32x4{T::low_float(w.x), T::high_float(w.x), T::low_float(w.y), T::high_float(w.y)};
  }
}

// PAST: past the caches.
template <class T, bool PAST>
__device__ inline void put4(typename T::storage* p, f32x4 x, bool vec) {
  if (vec) {
    if constexpr (!PAST)
      T::store4(p, x);
    else if constexpr (sizeof(typename T::storage) == 2)
      __builtin_nontemporal_store(u32x2{T::pack2(x.x, x.y), T::pack2(x.z, x.w)}, reinterpret_cast<u32x2*>(p));
    else
      __builtin_nontemporal_store(x, reinterpret_cast<f32x4*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = T::from_float(x[i]);
  }
}

// LPR lanes have one head's row, 8 elements each: two runs of four, chosen so
// that a lane holds both elements of its pairs and no value crosses lanes but
// the sum of squares.  A wave has U sets of 64 / LPR heads of one token: its
// lanes' cosines, sines and weights serve U heads.
template <class T, int LPR, int U>
__global__ void __launch_bounds__(256)
norm_rope_kernel(RopeArgs a) {
  using S = typename T::storage;
  constexpr int RPW = kWave / LPR;  // heads of a wave at a time
  const int lane = threadIdx.x & 63;
  const int heads = a.hq + a.hkv;
  const int sets = (heads + RPW * U - 1) / (RPW * U);
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int64_t t = w / sets;
  if (t >= a.tokens) return;
  const int h0 = static_cast<int>(w - t * sets) * (RPW * U) + lane / LPR;
  const int l = lane % LPR;
  const bool in = 8 * l < a.d;
  const bool turned = 8 * l < a.rotary;
  const bool split = turned && !a.interleaved;
  const int ea = split ? 4 * l : 8 * l, eb = split ? a.rotary / 2 + 4 * l : 8 * l + 4;
  const int64_t pos = a.pos_is_int64 ? static_cast<const int64_t*>(a.positions)[t]
                                     : static_cast<int64_t>(static_cast<const int32_t*>(a.positions)[t]);
  const bool known = pos >= 0 && pos < a.table_rows;
  f32x4 cs{1, 1, 1, 1}, sn{0, 0, 0, 0};
  if (turned && known) {
    const float* row = a.table + pos * a.rotary + 4 * l;
    cs = *reinterpret_cast<const f32x4*>(row);
    sn = *reinterpret_cast<const f32x4*>(row + a.rotary / 2);
  }
  f32x4 xa[U], xb[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u * RPW;
    xa[u] = xb[u] = f32x4{0, 0, 0, 0};
    if (in && h < heads) {
      const S* x = h < a.hq ? static_cast<const S*>(a.q) + t * a.q_st + h * a.q_sh
                            : static_cast<const S*>(a.k) + t * a.k_st + (h - a.hq) * a.k_sh;
      xa[u] = load4<T>(x + ea, a.vec);
      xb[u] = load4<T>(x + eb, a.vec);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int h = h0 + u * RPW;
    const void* weight = h < a.hq ? a.q_weight : a.k_weight;
    if (weight) {
      float sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += xa[u][i] * xa[u][i] + xb[u][i] * xb[u][i];
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
      const float inv = 1.0f / sqrtf(sum / static_cast<float>(a.d) + a.eps);
      if (in) {
        const f32x4 wa = a.weight_f32 ? load4<F32>(static_cast<const float*>(weight) + ea, a.vec)
                                      : load4<T>(static_cast<const S*>(weight) + ea, a.vec);
        const f32x4 wb = a.weight_f32 ? load4<F32>(static_cast<const float*>(weight) + eb, a.vec)
                                      : load4<T>(static_cast<const S*>(weight) + eb, a.vec);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          xa[u][i] = xa[u][i] * inv * wa[i];
          xb[u][i] = xb[u][i] * inv * wb[i];
        }
      }
    }
    f32x4 ya = xa[u], yb = xb[u];
    if (split) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ya[i] = xa[u][i] * cs[i] - xb[u][i] * sn[i];
        yb[i] = xb[u][i] * cs[i] + xa[u][i] * sn[i];
      }
    } else if (turned) {
      ya = f32x4{xa[u].x * cs.x - xa[u].y * sn.x, xa[u].y * cs.x + xa[u].x * sn.x,
                 xa[u].z * cs.y - xa[u].w * sn.y, xa[u].w * cs.y + xa[u].z * sn.y};
      yb = f32x4{xb[u].x * cs.z - xb[u].y * sn.z, xb[u].y * cs.z + xb[u].x * sn.z,
                 xb[u].z * cs.w - xb[u].w * sn.w, xb[u].w * cs.w + xb[u].z * sn.w};
    }
    if (!known) ya = yb = f32x4{NAN, NAN, NAN, NAN};
    if (in && h < heads) {
      S* y = h < a.hq ? static_cast<S*>(a.q_out) + t * a.qo_st + h * a.qo_sh
                      : static_cast<S*>(a.k_out) + t * a.ko_st + (h - a.hq) * a.ko_sh;
      put4<T, (U > 1)>(y + ea, ya, a.vec);
      put4<T, (U > 1)>(y + eb, yb, a.vec);
    }
  }
}

template <class T, int LPR, int U>
static int launch_rope(const RopeArgs& a, hipStream_t s) {
  constexpr int per = kWave / LPR * U;
  const int64_t waves = a.tokens * ((a.hq + a.hkv + per - 1) / per);
  const int64_t groups = (waves + 3) / 4;
  if (groups > 0x7fffffff) return set_error(KVHOT_EUNSUPPORTED, "norm_rope: too many tokens");
  hipLaunchKernelGGL((norm_rope_kernel<T, LPR, U>), dim3(static_cast<uint32_t>(groups)), dim3(256), 0, s, a);
  return launch_status("norm_rope");
}

template <class T>
static int launch_rope(const RopeArgs& a, hipStream_t s) {
  // Outputs that pass the 8 L2s' 32 MiB: two sets of heads a wave, stored past
  // the caches (8192 tokens of 40 heads of 128, bf16, 168 MB, inputs in the last
  // cache: 35.0 us; one set and ordinary stores 41.2, two 37.5, five 39.8, five
  // past the caches 36.2; inputs from HBM: 44, three sets 47).  Below that what is stored is read soon, and one set gives more waves.
  const int64_t bytes = a.tokens * (a.hq + a.hkv) * a.d * static_cast<int64_t>(sizeof(typename T::storage));
  if (bytes >= (int64_t{32} << 20)) {
    if (a.d <= 64) return launch_rope<T, 8, 2>(a, s);
    if (a.d <= 128) return launch_rope<T, 16, 2>(a, s);
    if (a.d <= 256) return launch_rope<T, 32, 2>(a, s);
    return launch_rope<T, 64, 2>(a, s);
  }
  if (a.d <= 64) return launch_rope<T, 8, 1>(a, s);
  if (a.d <= 128) return launch_rope<T, 16, 1>(a, s);
  if (a.d <= 256) return launch_rope<T, 32, 1>(a, s);
  return launch_rope<T, 64, 1>(a, s);
}

}  // namespace kvhot

using namespace kvhot;

extern "C" int kvhot_norm_rope(const void* q, const int64_t q_strides[3], const void* k, const int64_t k_strides[3],
                               void* q_out, const int64_t q_out_strides[3], void* k_out, const int64_t k_out_strides[3],
                               const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                               const float* table, int64_t table_rows, int64_t rotary_dim, int interleaved,
                               const void* positions, int positions_are_int64, int64_t num_tokens, int64_t num_q_heads,
                               int64_t num_kv_heads, int64_t head_dim, int dtype, void* stream) {
  clear_error();
  const int64_t es = dtype_size(dtype);
  if (es == 0) return set_error(KVHOT_EINVAL, "norm_rope: bad dtype");
  if (num_tokens < 0 || num_q_heads < 0 || num_kv_heads < 0 || head_dim <= 0 || rotary_dim < 0 || table_rows < 0 ||
      rotary_dim > head_dim)
    return set_error(KVHOT_EINVAL, "norm_rope: bad sizes");
  if (head_dim % 8 != 0 || head_dim > 512 || rotary_dim % 8 != 0)
    return set_error(KVHOT_EUNSUPPORTED, "norm_rope: head_dim (up to 512) and rotary_dim must be multiples of 8");
  if (num_q_heads > (1 << 20) || num_kv_heads > (1 << 20) || rotary_dim * table_rows < 0)
    return set_error(KVHOT_EUNSUPPORTED, "norm_rope: sizes beyond the kernel's range");
  if (num_tokens == 0 || num_q_heads + num_kv_heads == 0) return 0;
  if ((num_q_heads && (!q || !q_out || !q_strides || !q_out_strides)) ||
      (num_kv_heads && (!k || !k_out || !k_strides || !k_out_strides)) || !positions ||
      (rotary_dim > 0 && table_rows > 0 && !table))
    return set_error(KVHOT_EINVAL, "norm_rope: null pointer");
  if ((q_weight || k_weight) && weight_dtype != dtype && weight_dtype != KVHOT_F32)
    return set_error(KVHOT_EINVAL, "norm_rope: weights must be fp32 or of the values' dtype");
  if (reinterpret_cast<uintptr_t>(table) % 16) return set_error(KVHOT_EINVAL, "norm_rope: misaligned table");
  RopeArgs a{};
  a.q = q;
  a.k = k;
  a.q_out = q_out;
  a.k_out = k_out;
  bool vec = true;
  const auto strides = [&](const void* p, const int64_t* s, int64_t heads, int64_t& st, int64_t& sh) {
    st = sh = 0;
    if (heads == 0) return true;
    st = s[0];
    sh = s[1];
    const int64_t unit = 4 * es;
    if (reinterpret_cast<uintptr_t>(p) % unit || st * es % unit || sh * es % unit) vec = false;
    return s[2] == 1 && reinterpret_cast<uintptr_t>(p) % es == 0;
  };
  if (!strides(q, q_strides, num_q_heads, a.q_st, a.q_sh) || !strides(k, k_strides, num_kv_heads, a.k_st, a.k_sh) ||
      !strides(q_out, q_out_strides, num_q_heads, a.qo_st, a.qo_sh) ||
      !strides(k_out, k_out_strides, num_kv_heads, a.ko_st, a.ko_sh))
    return set_error(KVHOT_EINVAL, "norm_rope: head_dim must be the innermost, unit-stride dim of aligned tensors");
  const int64_t ws = dtype_size(weight_dtype);
  for (const void* p : {q_weight, k_weight}) {
    if (p && reinterpret_cast<uintptr_t>(p) % ws) return set_error(KVHOT_EINVAL, "norm_rope: misaligned weights");
    if (p && reinterpret_cast<uintptr_t>(p) % (4 * ws)) vec = false;
  }
  a.q_weight = q_weight;
  a.k_weight = k_weight;
  a.weight_f32 = weight_dtype == KVHOT_F32;
  a.table = table;
  a.table_rows = rotary_dim > 0 ? table_rows : INT64_MAX;
  a.positions = positions;
  a.pos_is_int64 = positions_are_int64 ? 1 : 0;
  a.tokens = num_tokens;
  a.hq = static_cast<int32_t>(num_q_heads);
  a.hkv = static_cast<int32_t>(num_kv_heads);
  a.d = static_cast<int32_t>(head_dim);
  a.rotary = static_cast<int32_t>(rotary_dim);
  a.interleaved = interleaved ? 1 : 0;
  a.vec = vec ? 1 : 0;
  a.eps = eps;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case KVHOT_F32: return launch_rope<F32>(a, s);
    case KVHOT_F16: return launch_rope<F16>(a, s);
    default: return launch_rope<BF16>(a, s);
  }
}
