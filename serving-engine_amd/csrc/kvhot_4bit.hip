// A KV cache held in 4 bits: the append that quantises, the dense read back
// and paged attention over it.
//
// A value is stored as a code (a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6) of
// 4 bits, times 2^e with one e for 32 elements of a head: the microscaling
// format that gfx950 converts in one instruction for two values
// (v_cvt_scalef32_pk_*_fp4), in both directions, to nearest even.  e is the
// exponent of the group's largest magnitude less 2, one more where its
// significand is above 1.75: then no value is off by more than 2^e, half the
// distance of the two largest codes.  Every value that comes out is a finite
// number of the type (kScaleLo, kScaleHi); a group that holds an infinity or
// a NaN comes out as NaN, all 32 of it (scale byte 255).
//
// Each (16 tokens, kv head) is one record of 17 * D bytes:
//   [0, 8D)           K codes, token by token: byte b holds elements 2b, 2b + 1
//   [8D, 16D)         V codes, pair by pair: byte 16 p + t holds elements
//                     2p, 2p + 1 of token t
//   [16D, 16D + D/2)  K scales, group by group: token 4 a + b at 4 b + a
//   [.., 17D)         V scales, group by group, token by token
// K rows are the A operand of S^T = K Q^T as they lie.  V's are the A operand
// of O^T = V^T P^T, whose k index is the token: with a pair's 16 tokens in 16
// consecutive bytes, a lane loads those of 4 to 8 pairs at once and no V ever
// goes through LDS.  (Pairs of tokens in a byte would save the permutes after
// the conversion, but an append would then have to read and write a byte that
// another token shares.)  The scale orders put what one lane needs into one
// load.
#include "kvhot_internal.h"

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <type_traits>


namespace kvhot {

// Smallest and largest scale byte by dtype: half the smallest scale and six
// times the largest are finite, normal values of the type (fp16: 2^-24, its
// smallest value, and 49152).
static int scale_lo(int dtype) { return dtype == KVHOT_F16 ? 104 : 2; }
static int scale_hi(int dtype) { return dtype == KVHOT_F16 ? 140 : 252; }

static bool head_dim_4bit(int64_t d) { return d == 64 || d == 96 || d == 128 || d == 256; }

// The slot's record, token in it, or nullptr for a slot outside the pool.
struct Pool4 {
  char* base;
  int64_t block_stride;  // bytes
  int64_t num_slots;
  int32_t block_size, heads, rec;
};

__device__ inline char* record_of(const Pool4& p, int64_t slot, int head, int& token) {
  if (slot < 0 || slot >= p.num_slots) return nullptr;
  const int64_t b = slot / p.block_size;
  const int in = static_cast<int>(slot - b * p.block_size);
  token = in & 15;
  return p.base + b * p.block_stride + (static_cast<int64_t>(in >> 4) * p.heads + head) * p.rec;
}

// Eight values of x, as floats.
template <class T>
__device__ inline void load8(const typename T::storage* p, bool vec, float (&x)[8]) {
  if constexpr (sizeof(typename T::storage) == 2) {
    u32x4 w;
    if (vec) {
      w = *reinterpret_cast<const u32x4*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = static_cast<uint32_t>(p[2 * i]) | static_cast<uint32_t>(p[2 * i + 1]) << 16;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = T::low_float(w[i]);
      x[2 * i + 1] = T::high_float(w[i]);
    }
  } else {
    if (vec) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = a[i];
        x[4 + i] = b[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
  }
}

// The group's scale byte from a lane's share of it: lanes 16 apart hold 8 of its
// 32 values each.
__device__ inline uint32_t scale_byte(const float (&x)[8], uint32_t lo, uint32_t hi) {
  // As integers the magnitudes order like the floats, infinities and NaN on top.
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16, kWave)));
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32, kWave)));
  if (top >= 0x7f800000u) return 255;
  const int e = static_cast<int>(top >> 23) + ((top & 0x7fffffu) > 0x600000u ? 1 : 0) - 2;
  return static_cast<uint32_t>(min(max(e, static_cast<int>(lo)), static_cast<int>(hi)));
}

__device__ inline uint32_t quantise8(const float (&x)[8], uint32_t byte) {
  if (byte == 255) return 0;
  const float s = __uint_as_float(byte << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
  return w;
}

// ------------------------------------------------------------------ append --

// A wave has 16 tokens of one head of K or V, GW groups of 32 elements in turn: lane
// l has elements 8 (l / 16) on of token l % 16.  The 16 tokens of a prompt then lie
// in the same lines of V, whose bytes of one pair are 16 tokens apart: with a
// token's row in neighbouring lanes instead, 4152 tokens of 8 heads took 21 us, so
// 12.9 (22 MB, bound by its loads and 4-byte and 1-byte stores).
struct Unit4 {
  int64_t t;  // the lane's token
  int32_t head, group;
  bool value, there;
};

template <int GW>
__device__ inline Unit4 unit_of(int64_t tokens, int32_t heads, int32_t groups, int64_t units) {
  Unit4 u;
  int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  u.there = w < units;
  const int32_t sets = groups / GW;
  u.group = static_cast<int32_t>(w % sets) * GW;
  w /= sets;
  u.value = w & 1;
  w >>= 1;
  u.head = static_cast<int32_t>(w % heads);
  u.t = w / heads * 16 + (threadIdx.x & 15);
  u.there = u.there && u.t < tokens;
  return u;
}

template <class T, typename SlotT, int GW>
__global__ void __launch_bounds__(256)
append_4bit_kernel(const typename T::storage* __restrict__ key, const typename T::storage* __restrict__ value,
                   Pool4 pool, const SlotT* __restrict__ slots, int64_t tokens, int32_t groups, int64_t units,
                   int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh, int k_vec, int v_vec, uint32_t lo,
                   uint32_t hi) {
  const Unit4 u = unit_of<GW>(tokens, pool.heads, groups, units);
  const int l = (threadIdx.x & 63) >> 4, d = groups * 32;
  float x[GW][8];
  int tok = 0;
  char* rec = nullptr;
  if (u.there) {
    rec = record_of(pool, static_cast<int64_t>(slots[u.t]), u.head, tok);
    const typename T::storage* src = u.value ? value + u.t * v_st + u.head * v_sh : key + u.t * k_st + u.head * k_sh;
#pragma unroll
    for (int i = 0; i < GW; ++i) load8<T>(src + (u.group + i) * 32 + l * 8, u.value ? v_vec : k_vec, x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < GW; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = 0;
  }
#pragma unroll
  for (int i = 0; i < GW; ++i) {
    const uint32_t byte = scale_byte(x[i], lo, hi);  // (the lanes of a token are there or not together)
    const uint32_t w = quantise8(x[i], byte);
    if (!rec) continue;
    const int g = u.group + i;
    if (!u.value) {
      *reinterpret_cast<uint32_t*>(rec + tok * (d / 2) + g * 16 + l * 4) = w;
      if (l == 0) rec[16 * d + g * 16 + (tok & 3) * 4 + (tok >> 2)] = static_cast<char>(byte);
    } else {
      char* v = rec + 8 * d + g * 256 + l * 64 + tok;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[16 * j] = static_cast<char>(w >> (8 * j));
      if (l == 0) rec[16 * d + d / 2 + g * 16 + tok] = static_cast<char>(byte);
    }
  }
}

// -------------------------------------------------------------- dense read --

// Two values of a code byte, as T's storage type pair (16-bit) or floats.
template <class T, int I>
__device__ inline uint32_t pair16(uint32_t w, float s) {
  if constexpr (std::is_same<T, F16>::value)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, I));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, I));
}

// The eight codes of w, times the scale, as four packed pairs of M (BF16 or F16).
template <class M>
__device__ inline u32x4 codes8(uint32_t w, float s) {
  return u32x4{pair16<M, 0>(w, s), pair16<M, 1>(w, s), pair16<M, 2>(w, s), pair16<M, 3>(w, s)};
}

// A scale byte as a float whose exponent it is: the conversions look at nothing
// else of it (255 makes them return NaN), so byte i of a word takes one shift.
__device__ inline float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ inline float scale_in(uint32_t word, int i) {
  return __uint_as_float(i == 3 ? word >> 1 : word << (23 - 8 * i));
}

template <bool CACHED, class V>
__device__ inline void put(V x, void* p) {
  if constexpr (CACHED)
    *static_cast<V*>(p) = x;
  else
    __builtin_nontemporal_store(x, static_cast<V*>(p));
}

// A wave reads 16 slots of one head, K or V.  It writes whole rows, D / 8 lanes a
// row, past the caches; K's codes are read in that order too.  V's are read as the
// append writes them, tokens side by side, and change lanes in LDS.  Bound by HBM:
// 90k tokens of 8 heads of 128 (480 MB in all) 119 us; with 64-byte pieces of 16
// rows in a store instead 192, with ordinary stores 165 even from the caches.
// BLOCKS: into kv-interleaved blocks of 16 tokens at `key` instead, NaN as 0, and
// stored where the next kernel finds them.
template <class T, typename SlotT, int D, bool BLOCKS>
__global__ void __launch_bounds__(256)
read_4bit_kernel(Pool4 pool, const SlotT* __restrict__ slots, int64_t tokens, int64_t units,
                 typename T::storage* __restrict__ key, typename T::storage* __restrict__ value) {
  constexpr int CH = D / 8, NI = D / 32;  // 8-element chunks of a row; chunks of a lane
  __shared__ uint32_t codes[4][16 * (CH + 1)];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t u = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  const bool there = u < units;  // (every wave meets the barrier)
  const bool is_v = u & 1;
  u >>= 1;
  const int head = static_cast<int>(u % pool.heads);
  const int64_t t0 = u / pool.heads * 16;
  int tok = 0;
  const int64_t mine = t0 + (lane & 15);
  const char* rec = there && mine < tokens ? record_of(pool, static_cast<int64_t>(slots[mine]), head, tok) : nullptr;
  uint32_t w[NI], byte[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) w[i] = 0;
  if (is_v && rec) {
    const int l = lane >> 4;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const uint8_t* v = reinterpret_cast<const uint8_t*>(rec) + 8 * D + i * 256 + l * 64 + tok;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[i] |= static_cast<uint32_t>(v[16 * j]) << (8 * j);
    }
  }
  const uint64_t at = reinterpret_cast<uint64_t>(rec);
  const int lo = static_cast<int>(at), hi = static_cast<int>(at >> 32);
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int t = (i * 64 + lane) / CH, c = (i * 64 + lane) % CH;
    const uint64_t r = static_cast<uint64_t>(static_cast<uint32_t>(__shfl(hi, t, kWave))) << 32 |
                       static_cast<uint32_t>(__shfl(lo, t, kWave));
    const int tk = __shfl(tok, t, kWave);
    const char* p = reinterpret_cast<const char*>(r);
    byte[i] = 127;
    if (p && is_v) {
      byte[i] = static_cast<uint8_t>(p[16 * D + D / 2 + (c >> 2) * 16 + tk]);
    } else if (p) {
      w[i] = *reinterpret_cast<const uint32_t*>(p + tk * (D / 2) + c * 4);
      byte[i] = static_cast<uint8_t>(p[16 * D + (c >> 2) * 16 + (tk & 3) * 4 + (tk >> 2)]);
    }
  }
  uint32_t* own = codes[wave];
  if (is_v) {
#pragma unroll
    for (int i = 0; i < NI; ++i) own[(lane & 15) * (CH + 1) + i * 4 + (lane >> 4)] = w[i];
  }
  __syncthreads();
  if (is_v) {
#pragma unroll
    for (int i = 0; i < NI; ++i) w[i] = own[(i * 64 + lane) / CH * (CH + 1) + (i * 64 + lane) % CH];
  }
  typename T::storage* out = is_v ? value : key;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int t = (i * 64 + lane) / CH, c = (i * 64 + lane) % CH;
    if (!there || t0 + t >= tokens) continue;
    typename T::storage* o = BLOCKS ? key + ((t0 / 16 * pool.heads + head) * 2 + (is_v ? 1 : 0)) * (16 * D) + t * D + c * 8
                                    : out + ((t0 + t) * pool.heads + head) * D + c * 8;
    if (BLOCKS && byte[i] == 255) {
      byte[i] = 127;
      w[i] = 0;
    }
    const float s = scale_of(byte[i]);
    if constexpr (std::is_same<T, F32>::value) {
      const u32x4 x = codes8<BF16>(w[i], s);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        put<BLOCKS>(f32x4{BF16::low_float(x[2 * h]), BF16::high_float(x[2 * h]), BF16::low_float(x[2 * h + 1]),
                          BF16::high_float(x[2 * h + 1])},
                    o + 4 * h);
    } else {
      put<BLOCKS>(codes8<T>(w[i], s), o);
    }
  }
}

// Groups of a wave: a whole head where there are many tokens (a wave then has
// its loads in flight together), one where there are few.
static int groups_a_wave(int64_t tokens, int64_t d) { return tokens >= 512 ? static_cast<int>(d == 256 ? 4 : d / 32) : 1; }

// --------------------------------------------------------------- attention --

struct Attn4Args {
  const void* q;
  int64_t q_st, q_sh;
  const char* cache;
  int64_t block_stride;
  void* out;
  int64_t o_st, o_sh;
  float* lse;
  int64_t l_st, l_sh;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t *q_lens, *k_lens, *q_starts, *q_offs;
  int64_t total_query;
  int32_t num_rows, hq, hkv, group, block_size, num_blocks, causal;
  float scale;     // |scale| * log2(e)
  int32_t negate;  // the scale is negative: Q's sign is turned
  int32_t q_vec;
  // the grid
  int32_t flat, parts, part_steps, max_q, max_k, spb;
  float* ws_o;
  float* ws_lse;
};

constexpr int kStep = 64;   // keys a wave attends at a time: four records
constexpr int kWaves4 = 4;  // most waves of a work-group, which share out its steps

// One query block of one row and kv head: 16 * MT (query, head) pairs, "m-rows",
// in the order query by query, against the key steps [step0, step1).
struct Block4 {
  int32_t row, head, first;  // first m-row
  int32_t rows;              // m-rows that exist
  int32_t q0, off;           // first query token of the row, its position
  int32_t k_len;
  int32_t limit;             // keys that any of the m-rows sees
  int32_t least;             // keys that all of them see
};

__device__ inline int imin(int a, int b) { return a < b ? a : b; }
__device__ inline int imax(int a, int b) { return a > b ? a : b; }

// The keys that m-row m of the row sees.
__device__ inline int sees(const Attn4Args& a, const Block4& b, int m) {
  if (!a.causal) return b.k_len;
  const int64_t s = static_cast<int64_t>(b.off) + m / a.group + 1;
  return static_cast<int>(s < 0 ? 0 : s < b.k_len ? s : b.k_len);
}

template <int ROWS>
__device__ inline bool block_of(const Attn4Args& a, int row, int head, int qb, Block4& b) {
  b.row = row;
  b.head = head;
  const int n_q = imin(a.q_lens[row], a.max_q);
  b.first = qb * ROWS;
  const int64_t all = static_cast<int64_t>(n_q) * a.group;
  if (n_q <= 0 || b.first >= all) return false;
  b.rows = static_cast<int>(all - b.first < ROWS ? all - b.first : ROWS);
  b.q0 = a.q_starts[row];
  b.off = a.q_offs[row];
  b.k_len = imin(imax(a.k_lens[row], 0), a.max_k);
  // (the table's columns bound what can be read)
  const int64_t held = a.bt_stride * a.block_size;
  if (b.k_len > held) b.k_len = static_cast<int>(held);
  b.limit = sees(a, b, b.first + b.rows - 1);
  b.least = sees(a, b, b.first);
  return true;
}

// Codes and scales of a step that a lane holds.
template <int D>
struct Keys4 {
  static constexpr int NJ = D / 32;
  uint32_t code[4][NJ];  // token 4 t + (lane & 3) of record (lane & 15) / 4, elements 8 * NJ * (lane / 16) on
  uint32_t scale[2];     // one byte for each t: of the first and the last element's group
};
template <int D>
struct Values4 {
  u32x4 code[D / 32];             // the 16 tokens of record lane / 16, pairs pair_of(lane & 15, c)
  u32x4 scale[D == 96 ? 3 : 1];   // theirs
};

// Pair of elements c of A row i of O^T's tiles.  At head_dim 96 an i has one
// pair in each group, otherwise all of an i's pairs lie in one.
template <int D>
__device__ constexpr int pair_of(int i, int c) { return D == 96 ? i + 16 * c : (D / 32) * i + c; }

// Where a lane's records of a step lie: the block ids come first, so that they
// can be asked for a step ahead.
struct Where4 {
  int32_t k_id, v_id, k_in, v_in;  // block, record in it
};

__device__ inline Where4 where(const Attn4Args& a, const Block4& b, int step, int lane) {
  const int last = (b.limit + 15) / 16 - 1;
  const int ks = imin(step * 4 + ((lane & 15) >> 2), last), vs = imin(step * 4 + (lane >> 4), last);
  const int32_t* bt = a.bt + static_cast<int64_t>(b.row) * a.bt_stride;
  if (a.spb == 1) return Where4{bt[ks], bt[vs], 0, 0};
  const int kb = ks / a.spb, vb = vs / a.spb;
  return Where4{bt[kb], bt[vb], ks - kb * a.spb, vs - vb * a.spb};
}

template <int D>
__device__ inline const char* record_at(const Attn4Args& a, const Block4& b, int id, int in) {
  id = imin(imax(id, 0), a.num_blocks - 1);
  return a.cache + id * a.block_stride + (static_cast<int64_t>(in) * a.hkv + b.head) * (17 * D);
}

template <int D>
__device__ inline void load_keys(const Attn4Args& a, const Block4& b, const Where4& w, int lane, Keys4<D>& s) {
  constexpr int NJ = D / 32;
  const int i = lane & 15, g = lane >> 4;
  const char* kr = record_at<D>(a, b, w.k_id, w.k_in);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const char* p = kr + (4 * t + (i & 3)) * (D / 2) + g * (4 * NJ);
    if constexpr (NJ == 2) {
      *reinterpret_cast<u32x2*>(s.code[t]) = *reinterpret_cast<const u32x2*>(p);
    } else if constexpr (NJ == 3) {
#pragma unroll
      for (int j = 0; j < 3; ++j) s.code[t][j] = reinterpret_cast<const uint32_t*>(p)[j];
    } else {
#pragma unroll
      for (int j = 0; j < NJ; j += 4) *reinterpret_cast<u32x4*>(s.code[t] + j) = *reinterpret_cast<const u32x4*>(p + 4 * j);
    }
  }
  const int g0 = (g * NJ) >> 2, g1 = (g * NJ + NJ - 1) >> 2;
  s.scale[0] = *reinterpret_cast<const uint32_t*>(kr + 16 * D + g0 * 16 + (i & 3) * 4);
  s.scale[1] = s.scale[0];
  if constexpr (NJ == 3 || NJ == 8) s.scale[1] = *reinterpret_cast<const uint32_t*>(kr + 16 * D + g1 * 16 + (i & 3) * 4);
}

template <int D>
__device__ inline void load_values(const Attn4Args& a, const Block4& b, const Where4& w, int lane, Values4<D>& s) {
  const int i = lane & 15;
  const char* vr = record_at<D>(a, b, w.v_id, w.v_in);
#pragma unroll
  for (int c = 0; c < D / 32; ++c) s.code[c] = *reinterpret_cast<const u32x4*>(vr + 8 * D + pair_of<D>(i, c) * 16);
#pragma unroll
  for (int c = 0; c < (D == 96 ? 3 : 1); ++c)
    s.scale[c] = *reinterpret_cast<const u32x4*>(vr + 16 * D + D / 2 + (pair_of<D>(i, c) >> 4) * 16);
}

// Running state of a wave: O^T tiles (tile 2 c + e holds element e of pair c),
// and for its lane's m-row the reference that exponents are taken against, the
// score above which it moves, and the lane's share of the sum.
template <int D, int MT>
struct State4 {
  f32x4 o[MT][D / 16];
  float ref[MT], above[MT], sum[MT];
};

// A reference that moves goes this far below the score that moved it, and
// moves again when a score is kRoom above it: probabilities then stay within
// 2^kRoom (fp16's 65504 included), and those that matter are normal numbers of
// fp16.
constexpr float kBelow = 8.0f, kRoom = 15.0f;

template <class M, int NP>
__device__ inline void split_pair(float a, float b, uint32_t (&p)[NP]) {
#pragma unroll
  for (int n = 0; n < NP; ++n) {
    p[n] = M::pack2(a, b);
    if (n + 1 < NP) {
      a -= M::low_float(p[n]);
      b -= M::high_float(p[n]);
    }
  }
}

// Q^T of the block, as B operands: lane (n, g) has elements 8 (NJ * g + j) on of m-row
// n of each tile; and how many keys that sees.
template <class IO, class M, int NP, int D, int MT>
__device__ inline void load_queries(const Attn4Args& a, const Block4& b, int lane, u32x4 (&q)[MT][NP][D / 32],
                                    int (&lim)[MT]) {
  constexpr int NJ = D / 32;
  const int n = lane & 15, g = lane >> 4;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int at = 16 * m + n, mr = b.first + at;
    const bool there = at < b.rows;
    const int64_t tok = static_cast<int64_t>(b.q0) + mr / a.group;
    lim[m] = there ? sees(a, b, mr) : b.limit;
    const bool ok = there && tok >= 0 && tok < a.total_query;
    const typename IO::storage* src = static_cast<const typename IO::storage*>(a.q) +
                                      (ok ? tok * a.q_st + (b.head * a.group + mr % a.group) * a.q_sh : 0);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float x[8];
      if (ok) {
        load8<IO>(src + 8 * (NJ * g + j), a.q_vec, x);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0;
      }
      if (a.negate) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = -x[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[NP];
        split_pair<M, NP>(x[2 * i], x[2 * i + 1], w);
#pragma unroll
        for (int k = 0; k < NP; ++k) q[m][k][j][i] = w[k];
      }
    }
  }
}

template <int D, int MT>
__device__ inline void clear(State4<D, MT>& st) {
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    st.ref[m] = 0;
    st.above[m] = -INFINITY;
    st.sum[m] = 0;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) st.o[m][c] = f32x4{0, 0, 0, 0};
  }
}

// Writes the block's m-rows: to the outputs, or, of a block cut into parts, to the
// workspace (rows from w0 on).
template <class IO, int D, int MT>
__device__ inline void finish(const Attn4Args& a, const Block4& b, bool whole, int64_t w0, int lane,
                              const State4<D, MT>& st) {
  const int n = lane & 15, g = lane >> 4;
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    float sum = st.sum[m];
    sum += __shfl_xor(sum, 16, kWave);
    sum += __shfl_xor(sum, 32, kWave);
    const int at = 16 * m + n, mr = b.first + at;
    if (at >= b.rows) continue;
    const float inv = sum == 0 ? 0.0f : 1.0f / sum;  // no key seen: 0
    const float lse2 = sum == 0 ? -INFINITY : st.ref[m] + F32::log2(sum);
    if (whole) {
      const int64_t tok = static_cast<int64_t>(b.q0) + mr / a.group;
      const int hd = b.head * a.group + mr % a.group;
      if (tok < 0 || tok >= a.total_query) continue;
      typename IO::storage* o = static_cast<typename IO::storage*>(a.out) + tok * a.o_st + hd * a.o_sh;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < D / 16; ++c) o[2 * pair_of<D>(4 * g + r, c >> 1) + (c & 1)] = IO::from_float(st.o[m][c][r] * inv);
      if (a.lse && g == 0) a.lse[tok * a.l_st + hd * a.l_sh] = lse2 * kLn2;
    } else {
      float* o = a.ws_o + (w0 + at) * D;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < D / 16; ++c) o[2 * pair_of<D>(4 * g + r, c >> 1) + (c & 1)] = st.o[m][c][r] * inv;
      if (g == 0) a.ws_lse[w0 + at] = lse2;
    }
  }
}

// S^T of a step: row 4 g + r of tile t is token 4 t + r of record g.  Q^T is
// q[tile][part][j]: element 8 (NJ * (lane / 16) + j) on of m-row lane & 15.
// (The barriers here and below keep the scheduler from converting everything
// first, for which there are no registers.)
template <class M, int NP, int D, int MT>
__device__ inline void scores(const Keys4<D>& s, const u32x4 (&q)[MT][NP][D / 32], int lane, f32x4 (&sc)[MT][4]) {
  constexpr int NJ = D / 32;
  const int g = lane >> 4;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int m = 0; m < MT; ++m) sc[m][t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const bool second = NJ == 8 ? j >= 4 : NJ == 3 ? ((g * 3 + j) >> 2) != ((g * 3) >> 2) : false;
      const uint32_t sw = second ? s.scale[1] : s.scale[0];
      const u32x4 k = codes8<M>(s.code[t][j], scale_in(sw, t));
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = NP - 1; n >= 0; --n) sc[m][t] = M::mfma(k, q[m][n][j], sc[m][t]);
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

__device__ inline float highest(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ inline float highest(f32x4 a, f32x4 b) {
  return highest(highest(highest(highest(a[0], a[1]), a[2]), highest(highest(a[3], b[0]), b[1])), highest(b[2], b[3]));
}

// Probabilities from scores: lane (n, g) holds m-row n's for the 16 keys first +
// key(t, r) (first the lane's, key(t, r) known here), the B operand of O^T's two products of 32 keys.  MASKED: some m-row does not see
// all 64 keys.
template <class M, int NP, int D, int MT, bool MASKED, class K>
__device__ inline void probabilities(f32x4 (&sc)[MT][4], const int (&sees)[MT], int first, K key, float scale,
                                     State4<D, MT>& st, u32x4 (&p)[MT][NP][2]) {
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    // (A NaN passes through IEEE's maximum, which needs no canonical operands, and
    // then moves nothing: what the m-row comes to is NaN by that score alone.)
    const int left = sees[m] - first;
    if (MASKED) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (key(t, r) >= left) sc[m][t][r] = -INFINITY;
    }
    float top = highest(highest(sc[m][0], sc[m][1]), highest(sc[m][2], sc[m][3]));
    if (__any(top * scale > st.above[m])) {
      top = __builtin_elementwise_maximum(top, __shfl_xor(top, 16, kWave));
      top = __builtin_elementwise_maximum(top, __shfl_xor(top, 32, kWave));
      if (top * scale > st.above[m]) {
        const float ref = top * scale - kBelow;
        const float f = st.above[m] == -INFINITY ? 0.0f : F32::exp2(st.ref[m] - ref);
        st.ref[m] = ref;
        st.above[m] = ref + kRoom;
        st.sum[m] *= f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r) st.o[m][c][r] *= f;
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        float x = BF16::exp2(fmaf(sc[m][t][r], scale, -st.ref[m])), y = BF16::exp2(fmaf(sc[m][t][r + 1], scale, -st.ref[m]));
        if (MASKED) {  // (a scale of 0 would make NaN of them)
          if (key(t, r) >= left) x = 0;
          if (key(t, r + 1) >= left) y = 0;
        }
        st.sum[m] += x + y;
        uint32_t w[NP];
        split_pair<M, NP>(x, y, w);
#pragma unroll
        for (int n = 0; n < NP; ++n) p[m][n][t >> 1][(t & 1) * 2 + (r >> 1)] = w[n];
      }
  }
}

// O^T += V^T P^T.
template <class M, int NP, int D, int MT, bool MASKED>
__device__ inline void weigh(const Values4<D>& s, const u32x4 (&p)[MT][NP][2], const int (&sees)[MT], int base, int limit,
                             int lane, State4<D, MT>& st) {
  constexpr int NJ = D / 32, NS = D == 96 ? 3 : 1;
  const int g = lane >> 4;
  // V's scales: one float a token.  In a masked step a NaN may belong to a key
  // that some m-row does not see, whose probability of 0 it would turn into NaN
  // too: it is taken out here and put into the m-rows that see it below.  What
  // lies behind the last key that any of them sees may be anything: its scales
  // are 1.
  u32x4 vs[NS];
  uint32_t bad[NS];
#pragma unroll
  for (int c = 0; c < NS; ++c) {
    vs[c] = s.scale[c];
    bad[c] = 0;
    if (MASKED) {
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        const uint32_t sh = 8 * (t & 3);
        const bool seen = t < limit - base - 16 * g, nan = ((vs[c][t >> 2] >> sh) & 255) == 255;
        if (seen && nan) bad[c] |= 1u << t;
        if (!seen || nan) vs[c][t >> 2] = (vs[c][t >> 2] & ~(255u << sh)) | 127u << sh;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    float f[NS][8];  // of tokens 8 u .. 8 u + 7
#pragma unroll
    for (int c = 0; c < NS; ++c)
#pragma unroll
      for (int t = 0; t < 8; ++t) f[c][t] = scale_in(vs[c][2 * u + (t >> 2)], t & 3);
#pragma unroll
    for (int c = 0; c < NJ; ++c) {
      u32x4 lo, hi;  // elements 2 pair, 2 pair + 1 of tokens 8 u .. 8 u + 7
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t code = s.code[c][2 * u + w];
        const float* x = f[NS == 3 ? c : 0] + 4 * w;
        const uint32_t a0 = pair16<M, 0>(code, x[0]), a1 = pair16<M, 1>(code, x[1]), a2 = pair16<M, 2>(code, x[2]),
                       a3 = pair16<M, 3>(code, x[3]);
        lo[2 * w] = __builtin_amdgcn_perm(a1, a0, 0x05040100);
        lo[2 * w + 1] = __builtin_amdgcn_perm(a3, a2, 0x05040100);
        hi[2 * w] = __builtin_amdgcn_perm(a1, a0, 0x07060302);
        hi[2 * w + 1] = __builtin_amdgcn_perm(a3, a2, 0x07060302);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = NP - 1; n >= 0; --n) {
          st.o[m][2 * c] = M::mfma(lo, p[m][n][u], st.o[m][2 * c]);
          st.o[m][2 * c + 1] = M::mfma(hi, p[m][n][u], st.o[m][2 * c + 1]);
        }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if constexpr (MASKED) {
    bool any = false;
#pragma unroll
    for (int c = 0; c < NS; ++c) any |= bad[c] != 0;
    if (__any(any)) {
      // How many NaN of its elements each m-row sees, as one more product.
      const uint32_t one = M::pack2(1.0f, 1.0f);
#pragma unroll
      for (int c = 0; c < NS; ++c)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          f32x4 n{0, 0, 0, 0};
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            u32x4 x, y;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int t = 8 * u + 2 * w, key = base + 16 * g + t;
              x[w] = ((bad[c] >> t) & 1 ? one & 0xffffu : 0) | ((bad[c] >> (t + 1)) & 1 ? one & 0xffff0000u : 0);
              y[w] = (key < sees[m] ? one & 0xffffu : 0) | (key + 1 < sees[m] ? one & 0xffff0000u : 0);
            }
            n = M::mfma(x, y, n);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (n[r] > 0) {
#pragma unroll
              for (int e = 0; e < D / 16; ++e)
                if (NS == 1 || (e >> 1) == c) st.o[m][e][r] = __builtin_nanf("");
            }
        }
    }
  }
}

// Adds the state of another wave, read from LDS, to this wave's.
template <int D, int MT>
__device__ inline void join(State4<D, MT>& a, const float* lds, int lane) {
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const float* p = lds + m * (D / 16 * 4 + 3) * kWave + lane;
    const float ref = p[0], above = p[kWave], sum = p[2 * kWave];
    float fa = 1.0f, fb = 1.0f;
    if (above == -INFINITY) {  // no finite score there: its sums are 0, or NaN
      fb = 0.0f;
    } else if (a.above[m] == -INFINITY) {
      fa = 0.0f;
      a.ref[m] = ref;
      a.above[m] = above;
    } else if (ref > a.ref[m]) {
      fa = F32::exp2(a.ref[m] - ref);
      a.ref[m] = ref;
      a.above[m] = above;
    } else {
      fb = F32::exp2(ref - a.ref[m]);
    }
    a.sum[m] = a.sum[m] * fa + sum * fb;
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) a.o[m][c][r] = a.o[m][c][r] * fa + p[(3 + c * 4 + r) * kWave] * fb;
  }
}

template <int D, int MT>
__device__ inline void park(const State4<D, MT>& a, float* lds, int lane) {
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    float* p = lds + m * (D / 16 * 4 + 3) * kWave + lane;
    p[0] = a.ref[m];
    p[kWave] = a.above[m];
    p[2 * kWave] = a.sum[m];
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) p[(3 + c * 4 + r) * kWave] = a.o[m][c][r];
  }
}

template <int D, int MT>
constexpr int parked() { return MT * (D / 16 * 4 + 3) * kWave; }

// The sum of x over the wave's lanes up to this one.
__device__ inline int64_t lanes_sum(int64_t x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(x, o, kWave);
    if (lane >= o) x += y;
  }
  return x;
}

// The query block `flat` of all rows, the longest first: of up to 64 rows the one
// with the most keys, and its last block (causal blocks' work grows along a row).
// Of more rows each lane first sums a run of them, and the run that holds the block
// is looked through in order (1000 rows of 2-9 queries: 64 rows after 64 instead,
// sorted, 440 us).  (A grid of rows times the longest row's blocks would launch
// work-groups for blocks that are not there, at 8 ns each.)
template <int ROWS>
__device__ inline bool flat_block(const Attn4Args& a, int64_t flat, int& row, int& qb) {
  const int lane = threadIdx.x & 63;
  const auto blocks = [&](int r, int end) {
    const int64_t n = r < end ? static_cast<int64_t>(imin(a.q_lens[r], a.max_q)) * a.group : 0;
    return n > 0 ? (n + ROWS - 1) / ROWS : 0;
  };
  int first = 0, end = a.num_rows;
  const bool many = a.num_rows > 64;
  if (many) {
    const int per = (a.num_rows + 63) / 64;
    int64_t mine = 0;
    for (int j = 0; j < per; ++j) mine += blocks(lane * per + j, end);
    const int64_t ends = lanes_sum(mine);
    const uint64_t after = __ballot(ends > flat);
    if (!after) return false;
    const int at = __builtin_ctzll(after);
    flat -= __shfl(ends - mine, at, kWave);
    first = __builtin_amdgcn_readfirstlane(at * per);
    end = imin(end, first + per);
  }
  for (; first < end; first += 64) {
    int64_t mine = blocks(first + lane, end);
    int from = lane;
    if (!many) {
      const int keys = mine > 0 ? a.k_lens[lane] : -1;
      const uint64_t with = __ballot(mine > 0);
      int rank = 0;  // rows that come before the lane's
      for (uint64_t left = with; left; left &= left - 1) {
        const int other = __builtin_ctzll(left), k = __builtin_amdgcn_readlane(keys, other);
        rank += k > keys || (k == keys && other < lane) ? 1 : 0;
      }
      // (lanes without blocks go behind the others, in their order)
      if (mine == 0) rank = __popcll(with) + __popcll(~with & ((uint64_t{1} << lane) - 1));
      from = __builtin_amdgcn_ds_permute(rank * 4, lane);  // the row of rank `lane`
      mine = __shfl(mine, from, kWave);
    }
    const int64_t ends = lanes_sum(mine);
    const uint64_t after = __ballot(ends > flat);
    if (after) {
      const int at = __builtin_ctzll(after);
      row = __builtin_amdgcn_readfirstlane(first + __shfl(from, at, kWave));
      qb = __builtin_amdgcn_readfirstlane(static_cast<int>(__shfl(ends, at, kWave) - 1 - flat));
      return true;
    }
    flat -= __shfl(ends, 63, kWave);
  }
  return false;
}

// The row and query block of grid block u: one block a row where no row has more.
template <int ROWS>
__device__ inline bool grid_block(const Attn4Args& a, int64_t u, int& row, int& qb) {
  if (a.flat) return flat_block<ROWS>(a, u, row, qb);
  row = static_cast<int>(u);
  qb = 0;
  return true;
}

// Waves a SIMD that the registers of an instantiation are for.
constexpr int waves_per_simd(int np, int d, int mt) { return np == 3 ? (d == 256 ? 1 : 2) : d == 256 || mt == 2 ? 2 : 3; }

// Attention over the cache: O^T = V^T P^T and S^T = K Q^T on the matrix cores, from
// records that a wave loads straight into registers, with the running reference and
// sum of a softmax.  Bound by HBM where rows are long (16 rows of 32768 keys at
// 32 / 8 heads of 128: 106-110 us, 5.3 TB/s of 570 MB), by latency where they are
// short (7-8 us of 1001 keys: lengths, block ids, records, the waves' join).  A step
// is 64 keys so that a lane's probabilities are a whole record's; its phases are
// kept apart by scheduling barriers, without which the conversions of a step were
// all hoisted and one wave filled a SIMD (174 us).  Probabilities of 16-bit queries
// are rounded to the type for the product with V: half a step of each weight, as
// the output's own rounding; those of fp32 queries, and the queries, are three bf16
// values each, whose products with the codes are exact.
template <class IO, class M, int NP, int D, int MT>
__global__ void __launch_bounds__(64 * kWaves4) __attribute__((amdgpu_waves_per_eu(waves_per_simd(NP, D, MT))))
attn_4bit_kernel(Attn4Args a) {
  constexpr int NJ = D / 32, ROWS = 16 * MT;
  extern __shared__ float lds[];  // half of the waves' states
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = static_cast<int>(blockDim.x) >> 6;
  int64_t u = blockIdx.x;
  const int head = static_cast<int>(u % a.hkv);
  u /= a.hkv;
  const int part = static_cast<int>(u % a.parts);
  u /= a.parts;
  int row, qb;
  Block4 b;
  if (!grid_block<ROWS>(a, u, row, qb) || !block_of<ROWS>(a, row, head, qb, b)) return;
  const int steps = (b.limit + kStep - 1) / kStep;
  const int step0 = part * a.part_steps, step1 = imin(steps, step0 + a.part_steps);
  if (part > 0 && step0 >= steps) return;
  u32x4 q[MT][NP][NJ];
  int lim[MT];
  load_queries<IO, M, NP, D, MT>(a, b, lane, q, lim);
  State4<D, MT> st;
  clear(st);
  // A step's keys are loaded while the step before is weighed, its values while
  // its scores are computed; block ids two steps ahead.
  int s = step0 + wave;
  if (s < step1) {
    Keys4<D> keys;
    Values4<D> values;
    Where4 w = where(a, b, s, lane);
    load_keys<D>(a, b, w, lane, keys);
    load_values<D>(a, b, w, lane, values);
    w = where(a, b, imin(s + waves, step1 - 1), lane);
    const auto step = [&](auto masked) {
      constexpr bool MASKED = decltype(masked)::value;
      f32x4 sc[MT][4];
      scores<M, NP, D, MT>(keys, q, lane, sc);
      load_keys<D>(a, b, w, lane, keys);
      __builtin_amdgcn_sched_barrier(0);
      u32x4 p[MT][NP][2];
      const auto key = [](int t, int r) { return 4 * t + r; };
      probabilities<M, NP, D, MT, MASKED>(sc, lim, s * kStep + 16 * (lane >> 4), key, a.scale, st, p);
      __builtin_amdgcn_sched_barrier(0);
      weigh<M, NP, D, MT, MASKED>(values, p, lim, s * kStep, b.limit, lane, st);
      load_values<D>(a, b, w, lane, values);
      w = where(a, b, imin(s + 2 * waves, step1 - 1), lane);
      s += waves;
    };
    const int full = imin(step1, b.least / kStep);  // steps that every m-row sees whole
    while (s < full) step(std::false_type());
    while (s < step1) step(std::true_type());
  }
  // The waves' states, joined in LDS: the upper half into the lower until one is
  // left (of 4 waves 2 and 3 into 0 and 1, then 1 into 0).
  for (int half = waves / 2; half > 0; half >>= 1) {
    if (wave >= half && wave < 2 * half) park<D, MT>(st, lds + (wave - half) * parked<D, MT>(), lane);
    __syncthreads();
    if (wave < half) join<D, MT>(st, lds + wave * parked<D, MT>(), lane);
    __syncthreads();
  }
  if (wave != 0) return;

  const int64_t w = (u * a.parts + part) * a.hkv + head;
  finish<IO, D, MT>(a, b, steps <= a.part_steps, w * ROWS, lane, st);
}

// Joins the parts of the query blocks that were cut: WAVES (1 or 4) waves an m-row,
// each with a run of its parts, eight on their way at a time.  Bound by those loads'
// latency, 1.2 us for eight parts.
template <class IO, int D, int ROWS, int WAVES>
__global__ void __launch_bounds__(256)
merge_4bit_kernel(Attn4Args a) {
  constexpr int PER = (D + 63) / 64, AHEAD = 8, SETS = ROWS * WAVES / 4;  // work-groups of a block
  __shared__ float lds[WAVES == 4 ? 3 * (PER + 2) * kWave : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t u = blockIdx.x;
  const int set = static_cast<int>(u % SETS);
  u /= SETS;
  const int head = static_cast<int>(u % a.hkv);
  u /= a.hkv;
  int row, qb;
  Block4 b;
  const int m = WAVES == 4 ? set : set * 4 + wave;
  if (!grid_block<ROWS>(a, u, row, qb) || !block_of<ROWS>(a, row, head, qb, b) || m >= b.rows) return;
  const int steps = (b.limit + kStep - 1) / kStep;
  const int parts = (steps + a.part_steps - 1) / a.part_steps;
  const int mr = b.first + m;
  const int64_t tok = static_cast<int64_t>(b.q0) + mr / a.group;
  const int hd = b.head * a.group + mr % a.group;
  if (parts <= 1 || tok < 0 || tok >= a.total_query) return;
  const int64_t w0 = u * a.parts * a.hkv + head;
  const int run = WAVES == 4 ? (parts + 3) / 4 : parts, begin = WAVES == 4 ? imin(wave * run, parts) : 0;
  const int end = imin(begin + run, parts);
  float ref = -INFINITY, sum = 0, x[PER] = {};
  for (int p0 = begin; p0 < end; p0 += AHEAD) {
    float l[AHEAD], y[AHEAD][PER];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int p = imin(p0 + k, end - 1);
      const int64_t w = (w0 + static_cast<int64_t>(p) * a.hkv) * ROWS + m;
      l[k] = p0 + k < end ? a.ws_lse[w] : -INFINITY;
#pragma unroll
      for (int i = 0; i < PER; ++i) y[k][i] = i * 64 + lane < D ? a.ws_o[w * D + i * 64 + lane] : 0.0f;
    }
    float top = ref;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) top = l[k] > top || l[k] != l[k] ? l[k] : top;
    const float base = top == -INFINITY ? 0.0f : top;  // no key seen so far
    const float keep = F32::exp2(ref - base);
    ref = top;
    sum *= keep;
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] *= keep;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      if (p0 + k >= end) break;
      const float f = F32::exp2(l[k] - base);
      sum += f;
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] += f * y[k][i];
    }
  }
  if constexpr (WAVES == 4) {  // (the m-row, and so every return above, is the work-group's)
    if (wave > 0) {
      float* p = lds + (wave - 1) * (PER + 2) * kWave + lane;
      p[0] = ref;
      p[kWave] = sum;
#pragma unroll
      for (int i = 0; i < PER; ++i) p[(2 + i) * kWave] = x[i];
    }
    __syncthreads();
    if (wave > 0) return;
    float top = ref;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const float l = lds[k * (PER + 2) * kWave + lane];
      top = l > top || l != l ? l : top;
    }
    const float base = top == -INFINITY ? 0.0f : top, keep = F32::exp2(ref - base);
    ref = top;
    sum *= keep;
#pragma unroll
    for (int i = 0; i < PER; ++i) x[i] *= keep;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const float* p = lds + k * (PER + 2) * kWave + lane;
      const float f = F32::exp2(p[0] - base);
      sum += f * p[kWave];
#pragma unroll
      for (int i = 0; i < PER; ++i) x[i] += f * p[(2 + i) * kWave];
    }
  }
  const float inv = sum == 0 ? 0.0f : 1.0f / sum;
  typename IO::storage* o = static_cast<typename IO::storage*>(a.out) + tok * a.o_st + hd * a.o_sh;
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (i * 64 + lane < D) o[i * 64 + lane] = IO::from_float(x[i] * inv);
  if (a.lse && lane == 0) a.lse[tok * a.l_st + hd * a.l_sh] = sum == 0 ? -INFINITY : (ref + F32::log2(sum)) * kLn2;
}

// NaN of the cache into the outputs of the queries that see it, where an attention
// over finite copies of its values wrote them.  A work-group looks through
// kNanRecords records of a row and kv head: their scales are a seventeenth of them.
constexpr int kNanRecords = 64;

struct Nan4Args {
  Attn4Args a;
  const int32_t* rows;  // rows of the block table
};

template <class IO>
__global__ void __launch_bounds__(256)
spread_nan_4bit_kernel(Nan4Args n, int d) {
  const Attn4Args& a = n.a;
  __shared__ int32_t first[9];  // first key with a NaN: in K, in each group of V
  const int r = blockIdx.x / a.hkv, head = blockIdx.x % a.hkv;
  const int row = n.rows[r];
  const int64_t held = a.bt_stride * a.block_size;
  int k_len = imin(imax(a.k_lens[r], 0), a.max_k);
  if (k_len > held) k_len = static_cast<int>(held);
  if (threadIdx.x < 9) first[threadIdx.x] = INT32_MAX;
  __syncthreads();
  const int begin = static_cast<int>(blockIdx.y) * kNanRecords, end = imin(begin + kNanRecords, (k_len + 15) / 16);
  const int chunks = d / 16, groups = d / 32;  // 16-byte pieces: K's groups, then V's
  for (int u = static_cast<int>(threadIdx.x); u < (end - begin) * chunks; u += 256) {
    const int rec = begin + u / chunks, c = u % chunks;
    const int id = imin(imax(a.bt[static_cast<int64_t>(row) * a.bt_stride + rec / a.spb], 0), a.num_blocks - 1);
    const char* p = a.cache + id * a.block_stride +
                    (static_cast<int64_t>(rec % a.spb) * a.hkv + head) * (17 * d) + 16 * d + c * 16;
    const u32x4 x = *reinterpret_cast<const u32x4*>(p);
    for (int i = 0; i < 16; ++i) {
      if (((x[i >> 2] >> (8 * (i & 3))) & 255) != 255) continue;
      const int t = c < groups ? (i & 3) * 4 + (i >> 2) : i;
      if (rec * 16 + t < k_len) atomicMin(&first[c < groups ? 0 : 1 + c - groups], rec * 16 + t);
    }
  }
  __syncthreads();
  int any = INT32_MAX;
  for (int g = 0; g <= groups; ++g) any = imin(any, first[g]);
  if (any == INT32_MAX) return;
  const int n_q = imin(a.q_lens[r], a.max_q);
  for (int64_t i = threadIdx.x; i < static_cast<int64_t>(n_q) * a.group; i += 256) {
    const int64_t tok = static_cast<int64_t>(a.q_starts[r]) + i / a.group;
    const int h = head * a.group + static_cast<int>(i % a.group);
    const int64_t last = a.causal ? static_cast<int64_t>(a.q_offs[r]) + i / a.group : k_len - 1;
    if (tok < 0 || tok >= a.total_query) continue;
    typename IO::storage* o = static_cast<typename IO::storage*>(a.out) + tok * a.o_st + h * a.o_sh;
    for (int g = 0; g < groups; ++g)
      if (first[0] <= last || first[1 + g] <= last)
        for (int e = 0; e < 32; ++e) o[32 * g + e] = IO::from_float(__builtin_nanf(""));
    if (first[0] <= last && a.lse) a.lse[tok * a.l_st + h * a.l_sh] = __builtin_nanf("");
  }
}

constexpr int64_t kWholeSteps = 128;

// Split of a call: tiles of 16 m-rows of a query block, blocks (of all rows), waves
// of a work-group, parts, key steps of a part, and the workspace: partials, then
// their logarithms.
struct Split4 {
  int32_t mt, flat, waves, parts, part_steps;
  int64_t blocks, ws_bytes;
};

static Split4 split_4bit(int64_t rows, int64_t total, int64_t max_q, int64_t max_k, int64_t group, int64_t hkv, int64_t d,
                         int dtype) {
  Split4 s;
  const int64_t longest = max_q * group, steps = (max_k + kStep - 1) / kStep;
  // no more blocks than the call's queries fill, and one more for each row
  const auto blocks = [&](int64_t m) {
    return longest <= m ? rows : std::min(rows * ((longest + m - 1) / m), total * group / m + std::min(rows, total));
  };
  // Two tiles share a step's conversion, in registers for two waves a SIMD, not
  // three: from 1024 blocks of one on (bf16, head_dim 128, 32 / 8 heads, us with
  // one and two: 8 rows of 32 queries on 2048 keys 22 / 39, of 64 37 / 31, of 512
  // 225 / 186; 300 queries on 5000 keys 54 / 61; 2048 on 2048 82 / 73).
  s.mt = longest > 16 && dtype != KVHOT_F32 && d <= 128 && blocks(16) * hkv >= 1024 ? 2 : 1;
  s.flat = longest > 16 * s.mt;
  s.blocks = blocks(16 * s.mt);
  // Blocks that give each of 256 CUs two work-groups are left whole up to
  // kWholeSteps steps (64 rows of 128-2048 keys: 23.6 us, in two parts 25.7 and
  // a merge of 4.8); fewer are cut for four work-groups a CU, of which three
  // fit: rows are ragged, and the parts behind a short row's end are empty
  // (24 rows of up to 6000 keys: 24.2 us, 26.9 when cut for three).  Up to 128,
  // rows of many parts, for those that fit (us cut for four and for three: a row of
  // 32768 keys 17.9 / 15.2, 4 of 16384 26.0 / 22.1, 8 38.7 / 35.0, of 1000-16384
  // 24.6 / 22.4, 16 of 8192 38.3 / 34.5; 4 of 1000-16384 16.8 / 17.8).
  const int64_t n = std::max<int64_t>(s.blocks * hkv, 1);
  const int64_t fit = 256 * waves_per_simd(dtype == KVHOT_F32 ? 3 : 1, static_cast<int>(d), s.mt);
  const int64_t parts = n >= 512 ? 1 : n > 128 ? (1024 + n - 1) / n : std::max<int64_t>(fit / n, 1);
  // Where blocks of up to 16 steps fill the CUs' waves without it, a block is one
  // wave's or two's: a start and a join then serve more steps (us with 4 waves, 2
  // and 1; 256 rows of up to 128 keys 23.1 / 16.6 / 12.8, of up to 1024 49.4 / 46.7 /
  // 44.8, of up to 2048 74 / 80 / 78; 128 rows of up to 1024 30.9 / 26.7 / 30.4, of
  // up to 4096 80 / 80 / 99; 1000 rows of 2-9 queries 316 / 194 / 136).
  s.waves = steps > 16 || n < 768 ? kWaves4 : n < 1536 ? 2 : 1;
  // A part has a step a wave at least; rows of two steps a wave stay whole (a row
  // of 1001 keys in parts of two 11.1 us, of one 10.2, a merge of 2.5 in both).
  const int64_t few = steps <= 2 * kWaves4 ? 2 * kWaves4 : kWaves4;
  const int64_t per = std::min<int64_t>(std::max<int64_t>((steps + parts - 1) / parts, few), kWholeSteps);
  s.part_steps = static_cast<int32_t>(per);
  s.parts = static_cast<int32_t>(std::max<int64_t>((steps + per - 1) / per, 1));
  s.ws_bytes = s.parts > 1 ? n * s.parts * 16 * s.mt * (d + 1) * 4 : 0;
  return s;
}

}  // namespace kvhot

using namespace kvhot;

static int check_pool(const char* what, const void* cache, int64_t block_stride, int64_t heads, int64_t d,
                      int64_t block_size, int64_t num_blocks) {
  const std::string w(what);
  if (heads <= 0 || d <= 0 || block_size <= 0 || num_blocks < 0) return set_error(KVHOT_EINVAL, w + ": bad sizes");
  if (!head_dim_4bit(d)) return set_error(KVHOT_EUNSUPPORTED, w + ": head_dim must be 64, 96, 128 or 256");
  if (block_size % 16 != 0) return set_error(KVHOT_EUNSUPPORTED, w + ": block_size must be a multiple of 16");
  if (num_blocks > 0x7fffffff || block_size > (1 << 20) || heads > (1 << 16))
    return set_error(KVHOT_EUNSUPPORTED, w + ": sizes beyond the kernels' range");
  if (!cache && num_blocks > 0) return set_error(KVHOT_EINVAL, w + ": null pointer");
  if (reinterpret_cast<uintptr_t>(cache) % 16 || block_stride % 16)
    return set_error(KVHOT_EINVAL, w + ": the cache and its block stride must be multiples of 16 bytes");
  if (num_blocks > 1 && block_stride < block_size / 16 * heads * 17 * d)
    return set_error(KVHOT_EINVAL, w + ": blocks overlap");
  return 0;
}

static Pool4 pool_of(const void* cache, int64_t block_stride, int64_t heads, int64_t d, int64_t block_size,
                     int64_t num_blocks) {
  return Pool4{const_cast<char*>(static_cast<const char*>(cache)), block_stride, num_blocks * block_size,
               static_cast<int32_t>(block_size), static_cast<int32_t>(heads), static_cast<int32_t>(17 * d)};
}

static bool aligned(const void* p, int64_t es, int64_t unit, std::initializer_list<int64_t> strides) {
  if (reinterpret_cast<uintptr_t>(p) % unit) return false;
  for (int64_t s : strides)
    if (s * es % unit) return false;
  return true;
}

// GO(T, slot type, N) for this call's dtype and slots, N groups a wave or the head_dim.
#define KVHOT_FOR_GROUPS(GO, T, S) \
  switch (gw) {                    \
    case 1: GO(T, S, 1); break;    \
    case 2: GO(T, S, 2); break;    \
    case 3: GO(T, S, 3); break;    \
    default: GO(T, S, 4); break;   \
  }
#define KVHOT_FOR_DIMS(GO, T, S)   \
  switch (head_dim) {              \
    case 64: GO(T, S, 64); break;  \
    case 96: GO(T, S, 96); break;  \
    case 128: GO(T, S, 128); break; \
    default: GO(T, S, 256); break; \
  }
#define KVHOT_FOR_TYPES(GO, FOR)                          \
  switch (dtype * 2 + (slot_is_int64 ? 1 : 0)) {          \
    case KVHOT_F32 * 2: FOR(GO, F32, int32_t) break;      \
    case KVHOT_F32 * 2 + 1: FOR(GO, F32, int64_t) break;  \
    case KVHOT_F16 * 2: FOR(GO, F16, int32_t) break;      \
    case KVHOT_F16 * 2 + 1: FOR(GO, F16, int64_t) break;  \
    case KVHOT_BF16 * 2: FOR(GO, BF16, int32_t) break;    \
    default: FOR(GO, BF16, int64_t) break;                \
  }

extern "C" int kvhot_reshape_and_cache_4bit(
    const void* key, const int64_t key_strides[3], const void* value, const int64_t value_strides[3], void* cache,
    int64_t block_stride_bytes, const void* slot_mapping, int slot_is_int64, int64_t num_tokens, int64_t num_kv_heads,
    int64_t head_dim, int64_t block_size, int64_t num_blocks, int dtype, void* stream) {
  clear_error();
  const int64_t es = dtype_size(dtype);
  if (es == 0) return set_error(KVHOT_EINVAL, "reshape_and_cache_4bit: bad dtype");
  if (num_tokens < 0) return set_error(KVHOT_EINVAL, "reshape_and_cache_4bit: bad sizes");
  if (int e = check_pool("reshape_and_cache_4bit", cache, block_stride_bytes, num_kv_heads, head_dim, block_size, num_blocks))
    return e;
  if (num_tokens == 0 || num_blocks == 0) return 0;
  if (!key || !value || !slot_mapping || !key_strides || !value_strides)
    return set_error(KVHOT_EINVAL, "reshape_and_cache_4bit: null pointer");
  if (key_strides[2] != 1 || value_strides[2] != 1)
    return set_error(KVHOT_EINVAL, "reshape_and_cache_4bit: head_dim must be the innermost, unit-stride dim");
  if (reinterpret_cast<uintptr_t>(key) % es || reinterpret_cast<uintptr_t>(value) % es)
    return set_error(KVHOT_EINVAL, "reshape_and_cache_4bit: misaligned tensors");
  const int gw = groups_a_wave(num_tokens, head_dim);
  const int64_t units = (num_tokens + 15) / 16 * num_kv_heads * 2 * (head_dim / 32 / gw);
  if ((units + 3) / 4 > 0x7fffffff) return set_error(KVHOT_EUNSUPPORTED, "reshape_and_cache_4bit: too many tokens");
  const Pool4 pool = pool_of(cache, block_stride_bytes, num_kv_heads, head_dim, block_size, num_blocks);
  const int kv = aligned(key, es, 16, {key_strides[0], key_strides[1]});
  const int vv = aligned(value, es, 16, {value_strides[0], value_strides[1]});
#define KVHOT_LAUNCH(T, S, GW)                                                                                        \
  hipLaunchKernelGGL((append_4bit_kernel<T, S, GW>), dim3(static_cast<uint32_t>((units + 3) / 4)), dim3(256), 0,      \
                     static_cast<hipStream_t>(stream), static_cast<const T::storage*>(key),                           \
                     static_cast<const T::storage*>(value), pool, static_cast<const S*>(slot_mapping), num_tokens,    \
                     static_cast<int32_t>(head_dim / 32), units, key_strides[0], key_strides[1], value_strides[0],    \
                     value_strides[1], kv, vv, scale_lo(dtype), scale_hi(dtype))
  KVHOT_FOR_TYPES(KVHOT_LAUNCH, KVHOT_FOR_GROUPS)
#undef KVHOT_LAUNCH
  return launch_status("reshape_and_cache_4bit");
}

extern "C" int kvhot_read_cache_4bit(const void* cache, int64_t block_stride_bytes, const void* slots, int slot_is_int64,
                                     int64_t num_slots, int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                     int64_t num_blocks, void* key, void* value, int as_blocks, int dtype, void* stream) {
  clear_error();
  if (dtype_size(dtype) == 0) return set_error(KVHOT_EINVAL, "read_cache_4bit: bad dtype");
  if (num_slots < 0) return set_error(KVHOT_EINVAL, "read_cache_4bit: bad sizes");
  if (int e = check_pool("read_cache_4bit", cache, block_stride_bytes, num_kv_heads, head_dim, block_size, num_blocks))
    return e;
  if (num_slots == 0) return 0;
  if (!key || (!value && !as_blocks) || !slots) return set_error(KVHOT_EINVAL, "read_cache_4bit: null pointer");
  if (as_blocks && num_slots % 16 != 0)
    return set_error(KVHOT_EINVAL, "read_cache_4bit: blocks of slots that are no multiple of 16");
  if (reinterpret_cast<uintptr_t>(key) % 16 || reinterpret_cast<uintptr_t>(value) % 16)
    return set_error(KVHOT_EINVAL, "read_cache_4bit: misaligned tensors");
  const int64_t units = (num_slots + 15) / 16 * num_kv_heads * 2;
  if ((units + 3) / 4 > 0x7fffffff) return set_error(KVHOT_EUNSUPPORTED, "read_cache_4bit: too many slots");
  const Pool4 pool = pool_of(cache, block_stride_bytes, num_kv_heads, head_dim, block_size, num_blocks);
#define KVHOT_LAUNCH(T, S, D)                                                                                    \
  hipLaunchKernelGGL((as_blocks ? read_4bit_kernel<T, S, D, true> : read_4bit_kernel<T, S, D, false>),              \
                     dim3(static_cast<uint32_t>((units + 3) / 4)), dim3(256), 0,                                 \
                     static_cast<hipStream_t>(stream), pool, static_cast<const S*>(slots), num_slots, units,     \
                     static_cast<T::storage*>(key), static_cast<T::storage*>(value))
  KVHOT_FOR_TYPES(KVHOT_LAUNCH, KVHOT_FOR_DIMS)
#undef KVHOT_LAUNCH
  return launch_status("read_cache_4bit");
}

static int check_attention(int64_t rows, int64_t total, int64_t max_q, int64_t max_k, int64_t hq, int64_t hkv, int64_t d,
                           int dtype) {
  if (rows < 0 || total < 0 || max_q < 0 || max_k < 0 || hq <= 0 || hkv <= 0 || d <= 0)
    return set_error(KVHOT_EINVAL, "paged_attention_4bit: bad sizes");
  if (hq % hkv != 0) return set_error(KVHOT_EINVAL, "paged_attention_4bit: num_q_heads must be a multiple of num_kv_heads");
  if (dtype_size(dtype) == 0) return set_error(KVHOT_EINVAL, "paged_attention_4bit: bad dtype");
  if (!head_dim_4bit(d)) return set_error(KVHOT_EUNSUPPORTED, "paged_attention_4bit: head_dim must be 64, 96, 128 or 256");
  if (max_k > 0x7fffff00 || max_q > 0x7fffff00 || rows > 0x3fffffff || total > 0x7fffffff || hq > (1 << 16) || max_q * (hq / hkv) > 0x7fffff00)
    return set_error(KVHOT_EUNSUPPORTED, "paged_attention_4bit: sizes beyond the kernels' range");
  return 0;
}

extern "C" int64_t kvhot_paged_attention_4bit_workspace_bytes(int64_t num_rows, int64_t sum_q_lens, int64_t max_q_len,
                                                              int64_t max_k_len, int64_t num_q_heads,
                                                              int64_t num_kv_heads, int64_t head_dim, int dtype) {
  clear_error();
  if (int e = check_attention(num_rows, sum_q_lens, max_q_len, max_k_len, num_q_heads, num_kv_heads, head_dim, dtype))
    return e;
  if (num_rows == 0 || sum_q_lens == 0 || max_q_len == 0) return 0;
  return split_4bit(num_rows, sum_q_lens, max_q_len, max_k_len, num_q_heads / num_kv_heads, num_kv_heads, head_dim, dtype)
      .ws_bytes;
}

namespace {

template <class IO, class M, int NP, int D, int MT>
int launch_4bit(const Split4& sp, const Attn4Args& a, hipStream_t s) {
  const int64_t blocks = sp.blocks * a.hkv;
  if (blocks * std::max<int64_t>(sp.parts, 16 * MT) > 0x7fffffff)
    return set_error(KVHOT_EUNSUPPORTED, "paged_attention_4bit: too many work-groups");
  const size_t lds = static_cast<size_t>(sp.waves / 2) * parked<D, MT>() * sizeof(float);
  hipLaunchKernelGGL((attn_4bit_kernel<IO, M, NP, D, MT>), dim3(static_cast<uint32_t>(blocks * sp.parts)),
                     dim3(64 * static_cast<uint32_t>(sp.waves)), lds, s, a);
  if (int e = launch_status("paged_attention_4bit")) return e;
  if (sp.parts == 1) return 0;
  // Parts of more than one trip are four waves' (us with one and four: 86 parts 15.4 /
  // 5.6, 32 7.5 / 3.8, 24 6.6 / 4.2, 12 4.9 / 4.8; one trip, 6 parts of 192 blocks,
  // 5.4 / 8.0: the work-groups are four times as many).
  if (sp.parts > 8)
    hipLaunchKernelGGL((merge_4bit_kernel<IO, D, 16 * MT, 4>), dim3(static_cast<uint32_t>(blocks * (16 * MT))), dim3(256), 0,
                       s, a);
  else
    hipLaunchKernelGGL((merge_4bit_kernel<IO, D, 16 * MT, 1>), dim3(static_cast<uint32_t>(blocks * (4 * MT))), dim3(256), 0,
                       s, a);
  return launch_status("paged_attention_4bit merge");
}

template <class IO, class M, int NP, int D>
int launch_4bit(const Split4& sp, const Attn4Args& a, hipStream_t s) {
  if constexpr (NP == 1 && D <= 128)
    if (sp.mt == 2) return launch_4bit<IO, M, NP, D, 2>(sp, a, s);
  return launch_4bit<IO, M, NP, D, 1>(sp, a, s);
}

template <class IO, class M, int NP>
int launch_4bit(const Split4& sp, const Attn4Args& a, int64_t d, hipStream_t s) {
  switch (d) {
    case 64: return launch_4bit<IO, M, NP, 64>(sp, a, s);
    case 96: return launch_4bit<IO, M, NP, 96>(sp, a, s);
    case 128: return launch_4bit<IO, M, NP, 128>(sp, a, s);
    default: return launch_4bit<IO, M, NP, 256>(sp, a, s);
  }
}

}  // namespace

static Attn4Args args_4bit(const void* q, const int64_t* q_strides, const void* cache, int64_t block_stride_bytes, void* out,
                           const int64_t* out_strides, float* lse, const int64_t* lse_strides, const int32_t* block_table,
                           int64_t bt_row_stride, const int32_t* q_lens, const int32_t* k_lens, const int32_t* q_starts,
                           const int32_t* q_pos_offsets, int64_t num_rows, int64_t total_query, int64_t max_q_len,
                           int64_t max_k_len, int64_t num_q_heads, int64_t num_kv_heads, int64_t block_size,
                           int64_t num_blocks, float scale, int attn_flags, int dtype) {
  const int64_t es = dtype_size(dtype);
  Attn4Args a{};
  a.q = q;
  a.q_st = q ? q_strides[0] : 0;
  a.q_sh = q ? q_strides[1] : 0;
  a.cache = static_cast<const char*>(cache);
  a.block_stride = block_stride_bytes;
  a.out = out;
  a.o_st = out_strides[0];
  a.o_sh = out_strides[1];
  a.lse = lse;
  a.l_st = lse ? lse_strides[0] : 0;
  a.l_sh = lse ? lse_strides[1] : 0;
  a.bt = block_table;
  a.bt_stride = bt_row_stride;
  a.q_lens = q_lens;
  a.k_lens = k_lens;
  a.q_starts = q_starts;
  a.q_offs = q_pos_offsets;
  a.total_query = total_query;
  a.num_rows = static_cast<int32_t>(num_rows);
  a.hq = static_cast<int32_t>(num_q_heads);
  a.hkv = static_cast<int32_t>(num_kv_heads);
  a.group = a.hq / a.hkv;
  a.block_size = static_cast<int32_t>(block_size);
  a.num_blocks = static_cast<int32_t>(num_blocks);
  a.causal = attn_flags & KVHOT_CAUSAL;
  a.scale = std::fabs(scale) * kLog2e;
  a.negate = scale < 0;
  a.q_vec = aligned(q, es, 16, {a.q_st, a.q_sh});
  a.max_q = static_cast<int32_t>(max_q_len);
  a.max_k = static_cast<int32_t>(max_k_len);
  a.spb = a.block_size / 16;
  return a;
}

extern "C" int kvhot_spread_nan_4bit(const void* cache, int64_t block_stride_bytes, void* out, const int64_t out_strides[3],
                                     float* lse, const int64_t lse_strides[2], const int32_t* block_table,
                                     int64_t bt_row_stride, const int32_t* rows, const int32_t* q_lens,
                                     const int32_t* k_lens, const int32_t* q_starts, const int32_t* q_pos_offsets,
                                     int64_t num_rows, int64_t total_query, int64_t max_q_len, int64_t max_k_len,
                                     int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
                                     int64_t num_blocks, int attn_flags, int dtype, void* stream) {
  clear_error();
  if (int e = check_attention(num_rows, total_query, max_q_len, max_k_len, num_q_heads, num_kv_heads, head_dim, dtype))
    return e;
  if (int e = check_pool("spread_nan_4bit", cache, block_stride_bytes, num_kv_heads, head_dim, block_size, num_blocks))
    return e;
  if (attn_flags & ~KVHOT_CAUSAL) return set_error(KVHOT_EINVAL, "spread_nan_4bit: unknown attn_flags");
  if (num_rows == 0 || total_query == 0 || max_q_len == 0 || max_k_len == 0 || num_blocks == 0) return 0;
  if (!out || !out_strides || (lse && !lse_strides) || !block_table || !rows || !q_lens || !k_lens || !q_starts || !q_pos_offsets)
    return set_error(KVHOT_EINVAL, "spread_nan_4bit: null pointer");
  if (out_strides[2] != 1 || bt_row_stride <= 0) return set_error(KVHOT_EINVAL, "spread_nan_4bit: bad strides");
  const int64_t y = ((max_k_len + 15) / 16 + kNanRecords - 1) / kNanRecords;
  if (num_rows * num_kv_heads > 0x7fffffff || y > 65535)
    return set_error(KVHOT_EUNSUPPORTED, "spread_nan_4bit: too many work-groups");
  Nan4Args n{args_4bit(nullptr, nullptr, cache, block_stride_bytes, out, out_strides, lse, lse_strides, block_table,
                       bt_row_stride, q_lens, k_lens, q_starts, q_pos_offsets, num_rows, total_query, max_q_len, max_k_len,
                       num_q_heads, num_kv_heads, block_size, num_blocks, 1.0f, attn_flags, dtype),
             rows};
  const dim3 grid(static_cast<uint32_t>(num_rows * num_kv_heads), static_cast<uint32_t>(y));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const int d = static_cast<int>(head_dim);
  switch (dtype) {
    case KVHOT_F32: hipLaunchKernelGGL(spread_nan_4bit_kernel<F32>, grid, dim3(256), 0, s, n, d); break;
    case KVHOT_F16: hipLaunchKernelGGL(spread_nan_4bit_kernel<F16>, grid, dim3(256), 0, s, n, d); break;
    default: hipLaunchKernelGGL(spread_nan_4bit_kernel<BF16>, grid, dim3(256), 0, s, n, d); break;
  }
  return launch_status("spread_nan_4bit");
}

extern "C" int kvhot_paged_attention_4bit(
    const void* q, const int64_t q_strides[3], const void* cache, int64_t block_stride_bytes, void* out,
    const int64_t out_strides[3], float* lse, const int64_t lse_strides[2], const int32_t* block_table,
    int64_t bt_row_stride, const int32_t* q_lens, const int32_t* k_lens, const int32_t* q_starts,
    const int32_t* q_pos_offsets, int64_t num_rows, int64_t total_query, int64_t sum_q_lens, int64_t max_q_len,
    int64_t max_k_len, int64_t num_q_heads, int64_t num_kv_heads, int64_t head_dim, int64_t block_size, int64_t num_blocks, float scale,
    int attn_flags, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (int e = check_attention(num_rows, total_query, max_q_len, max_k_len, num_q_heads, num_kv_heads, head_dim, dtype))
    return e;
  if (int e = check_pool("paged_attention_4bit", cache, block_stride_bytes, num_kv_heads, head_dim, block_size, num_blocks))
    return e;
  if (attn_flags & ~KVHOT_CAUSAL) return set_error(KVHOT_EINVAL, "paged_attention_4bit: unknown attn_flags");
  if (sum_q_lens < 0 || sum_q_lens > total_query) return set_error(KVHOT_EINVAL, "paged_attention_4bit: bad sum_q_lens");
  if (num_rows == 0 || sum_q_lens == 0 || max_q_len == 0) return 0;
  if (!q || !out || !q_strides || !out_strides || !q_lens || !k_lens || !q_starts || !q_pos_offsets ||
      (lse && !lse_strides) || (!block_table && bt_row_stride > 0 && max_k_len > 0))
    return set_error(KVHOT_EINVAL, "paged_attention_4bit: null pointer");
  if (q_strides[2] != 1 || out_strides[2] != 1)
    return set_error(KVHOT_EINVAL, "paged_attention_4bit: head_dim must be the innermost, unit-stride dim");
  if (bt_row_stride < 0) return set_error(KVHOT_EINVAL, "paged_attention_4bit: bad sizes");
  if (num_blocks == 0 && max_k_len > 0) return set_error(KVHOT_EINVAL, "paged_attention_4bit: keys but no blocks");
  const Split4 sp = split_4bit(num_rows, sum_q_lens, max_q_len, max_k_len, num_q_heads / num_kv_heads, num_kv_heads,
                               head_dim, dtype);
  if (sp.ws_bytes > 0 && (!workspace || workspace_bytes < sp.ws_bytes))
    return set_error(KVHOT_EWORKSPACE, "paged_attention_4bit: workspace missing or too small");
  Attn4Args a = args_4bit(q, q_strides, cache, block_stride_bytes, out, out_strides, lse, lse_strides, block_table,
                          bt_row_stride, q_lens, k_lens, q_starts, q_pos_offsets, num_rows, total_query, max_q_len, max_k_len,
                          num_q_heads, num_kv_heads, block_size, num_blocks, scale, attn_flags, dtype);
  a.flat = sp.flat;
  a.parts = sp.parts;
  a.part_steps = sp.part_steps;
  a.ws_o = static_cast<float*>(workspace);
  a.ws_lse = a.ws_o ? a.ws_o + sp.blocks * num_kv_heads * sp.parts * 16 * sp.mt * head_dim : nullptr;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case KVHOT_F32: return launch_4bit<F32, BF16, 3>(sp, a, head_dim, s);
    case KVHOT_F16: return launch_4bit<F16, F16, 1>(sp, a, head_dim, s);
    default: return launch_4bit<BF16, BF16, 1>(sp, a, head_dim, s);
  }
}
