// attention.hip -- causal attention of packed prompts (simp_rt_attention_packed_f32).
//
// out_i = sum_j p_ij v_j, p_i = softmax_j(scale q_i . k_j) over the keys j <= i +
// nk - nq of the row's sequence.  One pass over the keys with a running maximum m
// and sum l: o and l are scaled by e^(m_old - m_new) when a tile raises m.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

#include "serve_args.h"
#include "serve_device.h"

namespace simp {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));

struct PackedArgs {
  const float *q, *k, *v;
  float *out;
  const int *q_starts, *k_starts;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, o_row, o_head;  // strides
  int tq, tk, n, group, hs;
  float scale;
};

// Tile slots: sequence s has the slots starts[s] / R + s and on, R rows a tile: at most
// n / R + 1 of them for n rows, so the next one's begin behind.
template <int R>
__device__ __forceinline__ int seq_of_slot(const int *starts, int n, int rows, int t) {
  return last_of(n, [&](int s) { return clampi(starts[s], 0, rows) / R + s <= t; });
}

// The rows and keys of one sequence.
struct Seq {
  int qb, nq, kb, nk;  // first query row, queries, first key row, keys
};
__device__ __forceinline__ Seq seq_of(const PackedArgs &a, int s) {
  const int qb = clampi(a.q_starts[s], 0, a.tq), kb = clampi(a.k_starts[s], 0, a.tk);
  return Seq{qb, clampi(a.q_starts[s + 1], qb, a.tq) - qb, kb, clampi(a.k_starts[s + 1], kb, a.tk) - kb};
}

// Up to four values of a row from dimension d on, 0 past its end.
template <bool VEC>
__device__ __forceinline__ float4 load4(const float *row, int d, int hs) {
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (VEC) {
    if (d < hs) x = *(const float4 *)(row + d);
  } else {
    if (d < hs) x.x = row[d];
    if (d + 1 < hs) x.y = row[d + 1];
    if (d + 2 < hs) x.z = row[d + 2];
    if (d + 3 < hs) x.w = row[d + 3];
  }
  return x;
}

// ---- the fp32 form
//
// One wave's part of 16 queries of a head: the 16-key tiles from `from` on, `step`
// keys apart, into o, m and l (per lane group).  S^T = K Q^T on
// v_mfma_f32_16x16x4_f32 leaves a lane with the scores of keys 4g .. 4g+3 (g = lane /
// 16) for query lane % 16, the B operand of O^T += V^T P^T.  my: the last key that
// the lane's query sees; all: the last that every query of the 16 sees; last: the
// last that any does.  HB: 16-dimension blocks of a head.  VEC: rows are whole 16-byte
// chunks (head_size and strides multiples of 4, aligned pointers).
template <int HB, bool VEC>
__device__ __forceinline__ void attend16(const PackedArgs &a, const float *qr, const float *kp,
                                         const float *vp, int my, int all, int last, int from,
                                         int step, v4f (&o)[HB], float &m, float &l) {
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4, hs = a.hs;
  float4 q[HB];
#pragma unroll
  for (int j = 0; j < HB; j++) {
    q[j] = load4<VEC>(qr, 16 * j + 4 * g, hs);
    o[j] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  m = -INFINITY;
  l = 0.f;
  for (int key0 = from; key0 <= last; key0 += step) {
    float v[HB][4];  // V[key0 + 4g + r][16 j + r16]
    v4f sc = {0.f, 0.f, 0.f, 0.f};
    {
      const float *kr = kp + (int64_t)min(key0 + r16, last) * a.k_row;
#pragma unroll
      for (int j = 0; j < HB; j++) {
        const float4 k = load4<VEC>(kr, 16 * j + 4 * g, hs);
        sc = __builtin_amdgcn_mfma_f32_16x16x4f32(k.x, q[j].x, sc, 0, 0, 0);
        sc = __builtin_amdgcn_mfma_f32_16x16x4f32(k.y, q[j].y, sc, 0, 0, 0);
        sc = __builtin_amdgcn_mfma_f32_16x16x4f32(k.z, q[j].z, sc, 0, 0, 0);
        sc = __builtin_amdgcn_mfma_f32_16x16x4f32(k.w, q[j].w, sc, 0, 0, 0);
      }
    }
    bool odd = false;  // a value that 0 * v would not make 0
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const float *vr = vp + (int64_t)min(key0 + 4 * g + r, last) * a.v_row;
#pragma unroll
      for (int j = 0; j < HB; j++) {
        v[j][r] = vr[min(16 * j + r16, hs - 1)];
        odd |= !(fabsf(v[j][r]) < INFINITY);
      }
    }
    float mt = -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      sc[r] = key0 + 4 * g + r <= my ? sc[r] * a.scale : -INFINITY;
      mt = fmaxf(mt, sc[r]);
    }
    {  // over the four groups of lanes that share the query
      float x = mt, y = mt;
      permlane16_swap(x, y);
      mt = fmaxf(x, y);
      x = y = mt;
      permlane32_swap(x, y);
      mt = fmaxf(x, y);
    }
    const float mn = fmaxf(m, mt), mu = mn == -INFINITY ? 0.f : mn;  // no key seen so far
    const float alpha = expf(m - mu);
    float p[4], pl = 0.f;
#pragma unroll
    for (int r = 0; r < 4; r++) {
      p[r] = expf(sc[r] - mu);
      pl += p[r];
    }
    m = mn;
    l = l * alpha + pl;
#pragma unroll
    for (int j = 0; j < HB; j++)
#pragma unroll
      for (int r = 0; r < 4; r++) o[j][r] *= alpha;
    if (key0 + 15 > all && __any(odd)) {
      // Some query does not see all 16 keys, and a product with a hidden infinity
      // or NaN would reach its row: one key at a time, added where it is seen.
      for (int kk = 0; kk < 16; kk++) {
        const float pr = kk & 2 ? (kk & 1 ? p[3] : p[2]) : (kk & 1 ? p[1] : p[0]);
        const float pk = __shfl(pr, (kk >> 2) * 16 + r16);
        const float *vr = vp + (int64_t)min(key0 + kk, last) * a.v_row;
        if (key0 + kk <= my)
#pragma unroll
          for (int j = 0; j < HB; j++)
#pragma unroll
            for (int r = 0; r < 4; r++)
              o[j][r] = fmaf(pk, vr[min(16 * j + 4 * g + r, hs - 1)], o[j][r]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < HB; j++)
#pragma unroll
        for (int r = 0; r < 4; r++)
          o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j][r], p[r], o[j], 0, 0, 0);
    }
  }
  float x = l, y = l;
  permlane16_swap(x, y);
  l = x + y;
  x = y = l;
  permlane32_swap(x, y);
  l = x + y;
}

// ---- the split form
//
// Both products on v_mfma_f32_32x32x16_f16.  A number x, scaled by a power of two to
// below 2^15, is hi + lo + r with hi = f16(x), lo = f16(x - hi) and |r| <= 2^-22 |x|, but
// 2^-25 at least, 2^-39 of the largest number in the scaling; x y is taken as hi hi + hi lo
// + lo hi, each product exact and each sum fp32, and lo lo <= 2^-22 |x y| left out.  In
// the 2-norm that is as close as an fp32 product (1.5e-7 to 6e-7 off 64 bits for 16 to 60000
// keys, torch's fp32 products and sums 1.1e-7 to 1.5e-6), at three times an f16 product's
// cost instead of the fp32 matrix instruction's sixteen.  What it does not keep is the
// bits of single channels of K and V 2^16 and more below the others of their stage.
// A stage is 32 keys of a kv head in the form of 1 KB operand fragments, in the order
// that the matrix instruction's lanes want them: K's hi and lo, 16 dimensions each, then
// V's, 16 keys by 32 dimensions each.  S^T = K Q^T leaves a lane with 16 keys of one
// query, which are the B operand of O^T += V^T P^T in the order that V's keys have
// there, so no weight moves between lanes.
//   attn_f16_k     a block of NW waves takes NW units (32 queries of one head) of one kv
//                  head, so that the query heads of a group share the stages, and
//                  walks them through LDS.  It makes them itself from K and V rows, or
//                  (STORED) fetches what attn_stages_k has made once for all blocks.
//   attn_stages_k  makes the stages.
//   attn_join_k    where there are few units the keys are split over several blocks; this
//                  joins what they leave.
// A block whose keys the split form does not serve (a value that is not finite, or sizes
// too far apart), and a wave whose queries it does not, compute their rows in fp32 instead
// (2048 tokens of 32 heads over 8, 128 wide, with a NaN in the last value and 1e30 in the
// first: 990 us for 151; with 1e9 in a channel of every query 1079).

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int kStageKeys = 32;
// A key that is smaller than the largest of its stage by more than this, or a stage that
// is smaller than the largest before it, would lie too low in the other's scaling (up
// to here 24 bits of it are kept), and a key that a query does not see would cost the
// query's row bits.
constexpr int kSpread = 14;
// O is kept in the scaling of the largest stage so far.  A row that sees only the first
// stages has a sum of 2^13 there or more, and 24 bits below its largest value stay above fp32's
// subnormals as long as the scaling does not rise by more than this behind its last key.
constexpr int kClimb = 64;
// What lies this far below the largest element of its query keeps 23 bits or fewer.
constexpr int kWide = 16;

struct F16Args {
  PackedArgs p;
  int hk;               // kv heads
  int blocks;           // of one kv head and one split
  int splits, chunk;    // of the keys: stages a split takes
  float *part;          // [splits, tq, heads, head_size], each divided by its sum; with splits > 1
  float2 *stat;         // [splits, tq, heads]: maximum and sum
  uint4 *frags;         // STORED: [slots, kv heads] stages, slots as of tiles of 32 keys
  float4 *scales;       // STORED: [kv heads, slots]: 1 / the scaling of K and of V (NaN: not
  int slots;            // served), the largest value of V's smallest key
};

// The exponent that brings a largest magnitude (its bits) into [2^14, 2^15); the
// smallest ones as far as a power of two goes.
__device__ __forceinline__ int lift(uint32_t top) {
  return top ? min(14 + 127 - (int)(top >> 23), 126) : 0;
}
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// The lanes' largest number of bits of a magnitude: floats in order, NaN above all.
__device__ __forceinline__ uint32_t bits_of(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
  const auto both = [](uint32_t a, float b) { return max(a, __float_as_uint(b)); };
  v = both(v, dpp_mov<kDppXor1>(__uint_as_float(v)));
  v = both(v, dpp_mov<kDppXor2>(__uint_as_float(v)));
  v = both(v, dpp_mov<kDppHalfMirror>(__uint_as_float(v)));
  v = both(v, dpp_mov<kDppMirror>(__uint_as_float(v)));
  float a = __uint_as_float(v), b = a;
  permlane16_swap(a, b);
  v = both(__float_as_uint(a), b);
  a = b = __uint_as_float(v);
  permlane32_swap(a, b);
  return both(__float_as_uint(a), b);
}

// x - h for the low and the high half of a pair of f16 (one instruction each; the compiler
// takes two)
__device__ __forceinline__ float rest_lo(h2 h, float x) {
  float r;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
  return r;
}
__device__ __forceinline__ float rest_hi(h2 h, float x) {
  float r;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
  return r;
}

__device__ __forceinline__ void split8(const float (&x)[8], h8 &hi, h8 &lo) {
  typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const h2 h = __builtin_convertvector((f2{x[e], x[e + 1]}), h2);
    const f2 r = {rest_lo(h, x[e]), rest_hi(h, x[e + 1])};
    const h2 l = __builtin_convertvector(r, h2);
    hi[e] = h[0], hi[e + 1] = h[1];
    lo[e] = l[0], lo[e + 1] = l[1];
  }
}
__device__ __forceinline__ void split4(const float4 &x, float by, uint2 *hi, uint2 *lo) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = {x.x * by, x.y * by}, b = {x.z * by, x.w * by};
  const h2 p = __builtin_convertvector(a, h2), q = __builtin_convertvector(b, h2);
  const f2 r = {rest_lo(p, a[0]), rest_hi(p, a[1])}, s = {rest_lo(q, b[0]), rest_hi(q, b[1])};
  *hi = make_uint2(__builtin_bit_cast(uint32_t, p), __builtin_bit_cast(uint32_t, q));
  *lo = make_uint2(__builtin_bit_cast(uint32_t, __builtin_convertvector(r, h2)),
                   __builtin_bit_cast(uint32_t, __builtin_convertvector(s, h2)));
}
__device__ __forceinline__ h8 split8(const float (&x)[8], float by, uint4 *hi, uint4 *lo) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; i++) y[i] = x[i] * by;
  h8 h, l;
  split8(y, h, l);
  *hi = __builtin_bit_cast(uint4, h);
  *lo = __builtin_bit_cast(uint4, l);
  return h;
}

// A wave's part of the making of a stage by four waves.  K: the eight keys from 8 w on,
// whole rows, four dimensions to a lane and 32 (128 bytes of a row) to a piece, so that a load
// takes whole cache lines; eight lanes share a key.  V: fragments f = NB i + db, 8 keys of one
// dimension to a lane.  Keys behind the sequence's last one repeat it: no query sees
// them.  So do dimensions behind a row's last one: q is 0 there, and O's are not stored.
// The lane's place in the stage is a 32-bit offset (the caller sees to strides below
// 2^23), so that a whole stage costs no address arithmetic.
__device__ __forceinline__ int v_key(int i, int h, int e) { return 16 * i + 8 * (e >> 2) + 4 * h + (e & 3); }
// The smallest head_size that NB serves.
constexpr int least_head(int nb) { return nb <= 4 ? 32 * nb - 31 : 32 * nb - 63; }
template <int NB, bool VEC>
struct KPart {
  int key, d;         // of the lane
  uint32_t ko;        // bytes
  uint32_t at;        // in a stage, bytes: of piece 0's hi
  __device__ __forceinline__ void init(const PackedArgs &a, int wave) {
    const int lane = threadIdx.x & 63, c = lane & 7;
    key = 8 * wave + (lane >> 3);
    d = 4 * c;
    ko = (uint32_t)key * (4u * (uint32_t)a.k_row);
    at = (uint32_t)((2 * (c >> 2)) * 1024 + (32 * (c >> 1 & 1) + key) * 16 + 8 * (c & 1));
  }
  // kp: the stage's first key; last: its last key's number in the stage
  __device__ __forceinline__ void load(const PackedArgs &a, const float *kp, int last, float4 (&k)[NB]) const {
    const uint32_t row = last >= kStageKeys - 1 ? ko : (uint32_t)min(key, last) * (4u * (uint32_t)a.k_row);
    const char *kb = (const char *)kp;
#pragma unroll
    for (int p = 0; p < NB; p++) {
      const bool sure = 32 * p + 32 <= least_head(NB);
      const uint32_t end = 4u * (uint32_t)(a.hs - (VEC ? 4 : 1)), x = 4u * (uint32_t)d + 128u * p;
      if (VEC) {
        k[p] = *(const float4 *)(kb + (row + (sure ? x : min(x, end))));
      } else {
        k[p].x = *(const float *)(kb + (row + min(x, end)));
        k[p].y = *(const float *)(kb + (row + min(x + 4, end)));
        k[p].z = *(const float *)(kb + (row + min(x + 8, end)));
        k[p].w = *(const float *)(kb + (row + min(x + 12, end)));
      }
    }
  }
  // The key's largest magnitude, its bits, in all of its lanes.
  __device__ __forceinline__ static uint32_t top(const float4 (&k)[NB]) {
    uint32_t t = 0;
#pragma unroll
    for (int p = 0; p < NB; p++)
      t = max(t, max(max(bits_of(k[p].x), bits_of(k[p].y)), max(bits_of(k[p].z), bits_of(k[p].w))));
    const auto both = [](uint32_t x, float y) { return max(x, __float_as_uint(y)); };
    t = both(t, dpp_mov<kDppXor1>(__uint_as_float(t)));
    t = both(t, dpp_mov<kDppXor2>(__uint_as_float(t)));
    return both(t, dpp_mov<kDppHalfMirror>(__uint_as_float(t)));
  }
  __device__ __forceinline__ void split(const float4 &k, int p, float by, void *stage) const {
    uint2 hi, lo;
    split4(k, by, &hi, &lo);
    char *dst = (char *)stage + (at + 4096u * p);
    *(uint2 *)dst = hi;
    *(uint2 *)(dst + 1024) = lo;
  }
};
template <int NB>
struct VPart {
  uint32_t vd, vo;  // bytes
  __device__ __forceinline__ void init(const PackedArgs &a, int f) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    vd = 4u * (uint32_t)min(32 * (f % NB) + (lane & 31), a.hs - 1);
    vo = (uint32_t)(4 * h) * (4u * (uint32_t)a.v_row) + vd;
  }
  __device__ __forceinline__ void load(const PackedArgs &a, const float *vp, int last, int f, float (&v)[8]) const {
    const int lane = threadIdx.x & 63, h = lane >> 5, i = f / NB;
    const char *vb = (const char *)vp;
    if (last >= kStageKeys - 1) {
      const char *vi = vb + (int64_t)(16 * i) * (4 * a.v_row);
#pragma unroll
      for (int e = 0; e < 8; e++) v[e] = *(const float *)(vi + (int64_t)v_key(0, 0, e) * (4 * a.v_row) + vo);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++)
        v[e] = *(const float *)(vb + ((uint32_t)min(v_key(i, h, e), last) * (4u * (uint32_t)a.v_row) + vd));
    }
  }
};

// The largest magnitude of eight numbers, its bits: positive ones are in order as signed
// integers, negative ones as unsigned ones, NaN above all.
__device__ __forceinline__ uint32_t top8(const float (&x)[8]) {
  int p = 0;
  uint32_t n = 0;
#pragma unroll
  for (int e = 0; e < 8; e++) {
    p = max(p, __float_as_int(x[e]));
    n = max(n, __float_as_uint(x[e]));
  }
  return max((uint32_t)p, n & 0x7fffffffu & (uint32_t)((int)n >> 31));
}

// The largest magnitude of each of a V part's eight keys over the 32 lanes that share
// them (one half of the wave), as bits of f16 of the scaled numbers (their hi): a lane has
// keys 2 (lane & 3) and the next one.
__device__ __forceinline__ uint32_t top_keys(h8 hi) {
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  typedef uint16_t s2 __attribute__((ext_vector_type(2)));
  u4 x = __builtin_bit_cast(u4, hi) & 0x7fff7fffu;
  const auto both = [](uint32_t a, uint32_t b) {
    const s2 p = __builtin_bit_cast(s2, a), q = __builtin_bit_cast(s2, b);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(p, q));
  };
  const auto from = [](uint32_t v, auto c) { return __float_as_uint(dpp_mov<decltype(c)::value>(__uint_as_float(v))); };
  const int lane = threadIdx.x & 63;
  const bool odd1 = lane & 1, odd2 = lane & 2;
  const uint32_t a = both(odd1 ? x[1] : x[0], from(odd1 ? x[0] : x[1], std::integral_constant<int, kDppXor1>()));
  const uint32_t b = both(odd1 ? x[3] : x[2], from(odd1 ? x[2] : x[3], std::integral_constant<int, kDppXor1>()));
  uint32_t c = both(odd2 ? b : a, from(odd2 ? a : b, std::integral_constant<int, kDppXor2>()));
  // lanes that have the same pair are those of the same lane & 3
  c = both(c, from(c, std::integral_constant<int, 0x124>()));  // row_ror:4
  c = both(c, from(c, std::integral_constant<int, kDppRor8>()));
  float u = __uint_as_float(c), v = u;
  permlane16_swap(u, v);
  return both(__float_as_uint(u), __float_as_uint(v));
}

// One stage.  NB: 32-dimension blocks of a head.  4096 keys of 8 heads, 128 wide: 17 us
// for 34 MB read and as many written, 3.9 TB/s; memory bounds it.
template <int NB, bool VEC>
__global__ void __launch_bounds__(256) attn_stages_k(const F16Args a) {
  __shared__ uint32_t key_s[2][32];  // each key's largest magnitude: K, V
  const PackedArgs &p = a.p;
  const int slot = blockIdx.x, hk = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int s = seq_of_slot<kStageKeys>(p.k_starts, p.n, p.tk, slot);
  const Seq z = seq_of(p, s);
  const int key0 = kStageKeys * (slot - (z.kb / kStageKeys + s));
  if (key0 < 0 || key0 >= z.nk) return;
  const int last = z.nk - 1 - key0;
  if (tid < 32) key_s[1][tid] = 0;
  __syncthreads();
  const float *kp = p.k + (int64_t)(z.kb + key0) * p.k_row + hk * p.k_head;
  const float *vp = p.v + (int64_t)(z.kb + key0) * p.v_row + hk * p.v_head;
  constexpr int CH = (2 * NB + 3) / 4;
  float4 k[NB];
  float v[CH][8];
  KPart<NB, VEC> kpart;
  kpart.init(p, wave);
  kpart.load(p, kp, last, k);
#pragma unroll
  for (int c = 0; c < CH; c++) {
    const int f = wave + 4 * c;
    if (f >= 2 * NB) break;
    VPart<NB> vpart;
    vpart.init(p, f);
    vpart.load(p, vp, last, f, v[c]);
  }
  key_s[0][kpart.key] = kpart.top(k);
#pragma unroll
  for (int c = 0; c < CH; c++) {
    const int f = wave + 4 * c;
    if (f >= 2 * NB) break;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      uint32_t u = bits_of(v[c][e]);  // over the 32 lanes of a key
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) u = max(u, (uint32_t)__shfl_xor((int)u, d));
      if ((lane & 31) == 0) atomicMax(&key_s[1][v_key(f / NB, lane >> 5, e)], u);
    }
  }
  __syncthreads();
  uint32_t kt = 0, vt = 0, kl = ~0u, vl = ~0u;  // largest, and smallest that is not 0
#pragma unroll 8
  for (int i = 0; i < 32; i++) {
    const uint32_t x = key_s[0][i], y = key_s[1][i];
    kt = max(kt, x), kl = min(kl, x - 1);
    vt = max(vt, y), vl = min(vl, y - 1);
  }
  kl++, vl++;  // (0 - 1 is the largest number: a key of zeros does not count)
  const int ek = lift(kt), ev = lift(vt);
  if (tid == 0) {
    const bool bad = max(kt, vt) >= 0x7f800000u || (kl && (int)(kt >> 23) - (int)(kl >> 23) > kSpread) ||
                     (vl && (int)(vt >> 23) - (int)(vl >> 23) > kSpread);
    a.scales[(int64_t)hk * a.slots + slot] = make_float4(power(-ek), bad ? NAN : vt ? power(-ev) : 0.f, 0.f, 0.f);
  }
  uint4 *out = a.frags + ((int64_t)slot * a.hk + hk) * (NB * 8 * 64);
#pragma unroll
  for (int i = 0; i < NB; i++) kpart.split(k[i], i, power(ek), out);
#pragma unroll
  for (int c = 0; c < CH; c++) {
    const int f = wave + 4 * c;
    if (f >= 2 * NB) break;
    split8(v[c], power(ev), out + (4 * NB + 2 * f) * 64 + lane, out + (4 * NB + 2 * f + 1) * 64 + lane);
  }
}

// What a row, or its part of a piece, is divided by.  A piece in which every score is -inf
// has the sum 0 and leaves zeros, for its weight in the row is 0 too; a whole row of
// such scores stays 0 / 0.
__device__ __forceinline__ float one_over(float l, int splits) {
  return splits > 1 && l == 0.f ? 0.f : 1.f / l;
}

// The blocks of one kv head: sequence s has ((q_starts[s] / 32 + s) G / NW) + s and on.
template <int NW>
__device__ __forceinline__ int first_block(const PackedArgs &a, int s) {
  return (int)(((int64_t)(clampi(a.q_starts[s], 0, a.tq) / 32 + s) * a.group) / NW) + s;
}

// The 32 queries of a head that wave w of a block takes (tile >= tiles: none).
struct Unit {
  int tile, head;
};
template <int NW>
__device__ __forceinline__ Unit unit_of(const PackedArgs &a, int block, int wave, int hk) {
  const int64_t u = (int64_t)block * NW + wave;  // of the sequence
  const int tile = (int)min(u / a.group, (int64_t)INT32_MAX);
  return Unit{tile, hk * a.group + (int)(u % a.group)};
}

// Where O takes more than half of the vector registers it lives in the accumulation
// registers: what scales it in vector ones has to put it back, or the compiler moves all of it
// both ways in every stage (1500 tokens of 16 heads over 4, 256 wide: 172 us, 160 with this).
template <int NB>
__device__ __forceinline__ void keep(v16f (&o)[NB]) {
  if constexpr (NB >= 6) {
#pragma unroll
    for (int d = 0; d < NB; d++) asm volatile("" : "+a"(o[d]));
  }
}

// One stage of one wave: S^T, weights and O^T.  f: what turns a product sum into a power
// of two; er: V's scaling over O's, a power 2^er <= 1; all: the last key that every
// query of the wave sees.  beside(ds): a part of other work, which goes between the
// products of S^T; behind: what follows them.
template <int NB, bool MADE, class Beside, class Behind>
__device__ __forceinline__ void stage(const h8 *frag, const h8 (&qh)[2 * NB], const h8 (&ql)[2 * NB],
                                      float f, int key0, int my, int all, int h, int er,
                                      v16f (&o)[NB], float &m, float &l, Beside beside, Behind behind) {
  v16f s;
#pragma unroll
  for (int r = 0; r < 16; r++) s[r] = 0.f;
  // Two fragments are read ahead of the products that use two others: under the other
  // waves' reads one alone comes later than three products take.
  constexpr int kReads = 0x100, kProducts = 0x008;
  if constexpr (MADE) {
    h8 k[3][2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      k[i][0] = frag[(2 * i) * 64];
      k[i][1] = frag[(2 * i + 1) * 64];
    }
#pragma unroll
    for (int ds = 0; ds < 2 * NB; ds++) {
      __builtin_amdgcn_sched_barrier(0);
      if (ds + 2 < 2 * NB) {
        k[(ds + 2) % 3][0] = frag[(2 * ds + 4) * 64];
        k[(ds + 2) % 3][1] = frag[(2 * ds + 5) * 64];
      }
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[ds % 3][0], qh[ds], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[ds % 3][0], ql[ds], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[ds % 3][1], qh[ds], s, 0, 0, 0);
      beside(ds);
    }
    __builtin_amdgcn_sched_barrier(0);
  } else {
    h8 k[2 * NB][2];
#pragma unroll
    for (int ds = 0; ds < 2 * NB; ds++) {
      k[ds][0] = frag[(2 * ds) * 64];
      k[ds][1] = frag[(2 * ds + 1) * 64];
    }
#pragma unroll
    for (int ds = 0; ds < 2 * NB; ds++) {
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[ds][0], qh[ds], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[ds][0], ql[ds], s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[ds][1], qh[ds], s, 0, 0, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kReads, 4, 0);
#pragma unroll
    for (int ds = 0; ds < 2 * NB; ds++) {
      __builtin_amdgcn_sched_group_barrier(kProducts, 3, 0);
      __builtin_amdgcn_sched_group_barrier(kReads, 2, 0);
    }
  }
  behind();
  if (key0 + kStageKeys - 1 > all) {  // some query does not see all of them
#pragma unroll
    for (int r = 0; r < 16; r++)
      s[r] = key0 + 8 * (r >> 2) + 4 * h + (r & 3) <= my ? s[r] * f : -INFINITY;
    f = 1.f;
  }
  float mt = s[0];
#pragma unroll
  for (int r = 1; r < 16; r++) mt = fmaxf(mt, s[r]);
  {
    float u = mt, v = mt;
    permlane32_swap(u, v);
    mt = fmaxf(u, v) * f;
  }
  // The maximum is raised only where a weight would pass 4: weights of 2^13 to the largest
  // one's 1 still fit f16 then.
  keep(o);
  if (__any(mt > m + 2.f)) {
    const float mn = fmaxf(m, mt), alpha = pow2(m - mn);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < NB; d++)
#pragma unroll
      for (int r = 0; r < 16; r++) o[d][r] *= alpha;
    keep(o);
  }
  keep(o);
  const float off = (float)(13 + er) - m;
  float pl = 0.f;
  {
    h8 ph[2], pw[2], v[2][NB][2];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int d = 0; d < NB; d++) {
        v[i][d][0] = frag[(4 * NB + 2 * (i * NB + d)) * 64];
        v[i][d][1] = frag[(4 * NB + 2 * (i * NB + d) + 1) * 64];
      }
#pragma unroll
    for (int i = 0; i < 2; i++) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        x[e] = pow2(fmaf(s[8 * i + e], f, off));
        pl += x[e];
      }
      split8(x, ph[i], pw[i]);
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int d = 0; d < NB; d++) {
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i][d][0], ph[i], o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i][d][0], pw[i], o[d], 0, 0, 0);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i][d][1], ph[i], o[d], 0, 0, 0);
      }
    __builtin_amdgcn_sched_group_barrier(kReads, 4, 1);
#pragma unroll
    for (int d = 0; d < 2 * NB; d++) {
      __builtin_amdgcn_sched_group_barrier(kProducts, 3, 1);
      __builtin_amdgcn_sched_group_barrier(kReads, 2, 1);
    }
  }
  l = fmaf(pl, power(-13 - er), l);
}

// NB: 32-dimension blocks; NW: waves; NS: stages in LDS.
// STORED, 4096 tokens of 32 heads over 8, 128 wide: 355 us, 1.16e15 f16 operations a second
// (a library's f16 product of 8192^3: 1.20e15); power bounds it (1.9 GHz), the matrix
// cores are busy 56 % of the time.  Four waves with two stages take 440 us: eight share what
// is fetched, and four stages hide the way of it.
// Made, 64 wide: a stage takes a block that has its CU alone 1.6 us, 0.35 of it products: its
// waves wait for themselves (the maximum, the exponentials, the stage's sizes).  Two
// groups of waves to a block, each with every other stage, take 2.9 us for two, and twice
// the registers: slower where the chip is full.  The loads behind the making of each
// part instead of behind all of them: the same.
template <int NB, int NW, int NS, bool VEC, bool STORED>
__global__ void __launch_bounds__(64 * NW, NB == 1 || (NB == 2 && STORED) ? 4 : NB == 2 ? 3 : NB <= 4 ? 2 : 1)
    attn_f16_k(const F16Args args) {
  constexpr int kFrags = 8 * NB, FPW = kFrags / NW;  // fragments of a stage; fetched by a wave
  constexpr int CH = (2 * NB + NW - 1) / NW;         // made by a wave, of K and of V
  static_assert(kFrags % NW == 0, "each wave fetches as many fragments");
  __shared__ uint4 ring[NS][kFrags * 64];
  __shared__ uint2 top_s[2][NW];
  __shared__ uint32_t key_s[3][2][32];  // each key's largest of a made stage
  const PackedArgs &a = args.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  // the last rows of a sequence, which see most keys, come first
  const int hk = blockIdx.x % args.hk, split = blockIdx.y;
  const int w = args.blocks - 1 - blockIdx.x / args.hk;
  const int seq = last_of(a.n, [&](int s) { return first_block<NW>(a, s) <= w; });
  const int block = w - first_block<NW>(a, seq);
  const Seq z = seq_of(a, seq);
  const int tiles = (z.nq + 31) / 32, off = z.nk - z.nq;
  const Unit un = unit_of<NW>(a, block, wave, hk);
  // the block's last key, and its stages
  const int top_tile = min(tiles - 1, unit_of<NW>(a, block, NW - 1, hk).tile);
  const int bend = min(32 * top_tile + 31, z.nq - 1) + off;
  const int st0 = split * args.chunk;
  const int st1 = min(bend < 0 ? 0 : bend / kStageKeys + 1, st0 + args.chunk);
  // (the last: attn_join_k reads nothing of it)
  if (block < 0 || unit_of<NW>(a, block, 0, hk).tile >= tiles || (split > 0 && st0 >= st1)) return;
  const bool idle = un.tile >= tiles;
  const int row0 = 32 * min(un.tile, tiles), row = min(row0 + r32, z.nq - 1);  // the lane's query
  const int my = row + off;                                     // its last key, or negative
  const int all = row0 + off;                                   // what every query sees
  const int wend = idle ? -1 : min(row0 + 31, z.nq - 1) + off;  // the wave's last key
  const int slot0 = z.kb / kStageKeys + seq;
  bool odd = false;

  // O's scaling over V's: the largest of the stages before (made), or of all (STORED)
  const float4 *scales = args.scales + (int64_t)hk * args.slots + slot0;
  int unit = -1000;
  if constexpr (STORED) {
    float hi = 0.f, lo = INFINITY;
    for (int i = threadIdx.x; i < (bend < 0 ? 0 : bend / kStageKeys + 1); i += 64 * NW) {
      const float v = scales[i].y;
      odd |= v != v;
      hi = fmaxf(hi, v);
      lo = fminf(lo, v > 0.f ? v : INFINITY);
    }
    hi = wave_max_dpp(hi);
    lo = -wave_max_dpp(-lo);
    if (lane == 0) top_s[0][wave] = make_uint2(__float_as_uint(hi), __float_as_uint(lo));
    odd = __syncthreads_or(odd);
#pragma unroll
    for (int i = 0; i < NW; i++) {
      hi = fmaxf(hi, __uint_as_float(top_s[0][i].x));
      lo = fminf(lo, __uint_as_float(top_s[0][i].y));
    }
    odd |= lo < hi * (1.f / (1 << kSpread));
    unit = (__float_as_int(hi) >> 23) - 127;
  }
  const float *kp = a.k + (int64_t)z.kb * a.k_row + hk * a.k_head;
  const float *vp = a.v + (int64_t)z.kb * a.v_row + hk * a.v_head;
  const uint32_t lds0 = lds_offset(&ring[0][0]);
  auto fetch = [&](int st) {
    const uint4 *src = args.frags + ((int64_t)(slot0 + st) * args.hk + hk) * (kFrags * 64) + lane;
    const uint32_t dst = lds0 + (uint32_t)((st - st0) % NS) * (kFrags * 1024);
#pragma unroll
    for (int i = 0; i < FPW; i++) {
      const int f = wave + i * NW;
      dma16(src + f * 64, dst + f * 1024);
    }
  };
  // (some waves repeat the last fragment)
  const auto frag_of = [&](int c) { return 2 * NB % NW ? min(wave + c * NW, 2 * NB - 1) : wave + c * NW; };
  float4 kx[NB];
  float vx[CH][8];
  uint32_t key_top;
  KPart<NB, VEC> kpart;
  VPart<NB> vpart[CH];
  if constexpr (!STORED) {
    kpart.init(a, wave);
#pragma unroll
    for (int c = 0; c < CH; c++) vpart[c].init(a, frag_of(c));
  }
  auto load = [&](int st) {
    const int key0 = kStageKeys * st, last = z.nk - 1 - key0;
    kpart.load(a, kp + (int64_t)key0 * a.k_row, last, kx);
#pragma unroll
    for (int c = 0; c < CH; c++) vpart[c].load(a, vp + (int64_t)key0 * a.v_row, last, frag_of(c), vx[c]);
  };
  // What is loaded: its largest magnitudes, for all waves; then in its fragments, with
  // the scalings 2^ek and 2^ev; then each key's largest, K's as it is, V's scaled.
  auto post = [&](int at) {
    uint32_t vt = 0;
    key_top = kpart.top(kx);
#pragma unroll
    for (int c = 0; c < CH; c++) vt = max(vt, top8(vx[c]));
    const uint32_t kt = wave_max_bits(key_top);
    vt = wave_max_bits(vt);
    if (lane == 0) top_s[at][wave] = make_uint2(kt, vt);
  };
  auto tops = [&](int at) {
    uint2 t = top_s[at][0];
#pragma unroll
    for (int i = 1; i < NW; i++) {
      t.x = max(t.x, top_s[at][i].x);
      t.y = max(t.y, top_s[at][i].y);
    }
    t.x = __builtin_amdgcn_readfirstlane(t.x);
    t.y = __builtin_amdgcn_readfirstlane(t.y);
    return t;
  };
  h8 v_hi[CH];
  auto make = [&](uint4 *dst, uint2 t, int part) {  // part: of 2 NB
    if (part % 2 == 0) {
      kpart.split(kx[part / 2], part / 2, power(lift(t.x)), dst);
    } else if (part / 2 < CH) {
      const int c = part / 2, f = frag_of(c);
      v_hi[c] = split8(vx[c], power(lift(t.y)), dst + (4 * NB + 2 * f) * 64 + lane, dst + (4 * NB + 2 * f + 1) * 64 + lane);
    }
  };
  auto key_tops = [&](int at) {
    key_s[at][0][kpart.key] = key_top;
#pragma unroll
    for (int c = 0; c < CH; c++) {
      const uint32_t t = top_keys(v_hi[c]);
      if ((r32 & ~3) == 0) {  // keys 2 (lane & 3) and the next of the half's eight
        uint32_t *key = &key_s[at][1][v_key(frag_of(c) / NB, h, 2 * (lane & 3))];
        atomicMax(key, t & 0xffffu);
        atomicMax(key + 1, t >> 16);
      }
    }
  };
  if constexpr (STORED) {
#pragma unroll
    for (int i = 0; i < NS - 1; i++)
      if (!odd && st0 + i < st1) fetch(st0 + i);
  } else if (st0 < st1) {
    load(st0);
    if (threadIdx.x < 32) key_s[0][1][r32] = key_s[1][1][r32] = 0;
  }

  h8 qh[2 * NB], ql[2 * NB];
  float qf;
  bool wide = false;  // some query of the wave spreads too far
  {
    const float *qr = a.q + (int64_t)(z.qb + row) * a.q_row + un.head * a.q_head;
    uint32_t top = 0;
    float x[2 * NB][8];
#pragma unroll
    for (int ds = 0; ds < 2 * NB; ds++) {
      const int d0 = 16 * ds + 8 * h;
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const float4 v = idle ? make_float4(0.f, 0.f, 0.f, 0.f) : load4<VEC>(qr, d0 + e, a.hs);
        x[ds][e] = v.x, x[ds][e + 1] = v.y, x[ds][e + 2] = v.z, x[ds][e + 3] = v.w;
      }
#pragma unroll
      for (int e = 0; e < 8; e++) top = max(top, bits_of(x[ds][e]));
    }
    {
      float u = __uint_as_float(top), v = u;
      permlane32_swap(u, v);
      top = max(__float_as_uint(u), __float_as_uint(v));
    }
    // A query half of whose elements lie far below its largest: one channel masks keys, say,
    // and the others, which decide, would keep few bits in its scaling.
    {
      const uint32_t limit = (uint32_t)max((int)top - (kWide << 23), 1) - 1;
      int low = 0;
#pragma unroll
      for (int ds = 0; ds < 2 * NB; ds++)
#pragma unroll
        for (int e = 0; e < 8; e++) low += bits_of(x[ds][e]) - 1 < limit;
      float u = __int_as_float(low), v = u;
      permlane32_swap(u, v);
      low = __float_as_int(u) + __float_as_int(v);
      wide = __any(2 * low >= a.hs);
    }
    const int eq = top < 0x7f800000u ? lift(top) : 0;  // infinities and NaN come through
    const float sign = a.scale < 0.f ? -1.f : 1.f;
    qf = ldexpf(fabsf(a.scale) * 1.44269504f, -eq);
#pragma unroll
    for (int ds = 0; ds < 2 * NB; ds++) {
#pragma unroll
      for (int e = 0; e < 8; e++) x[ds][e] = ldexpf(sign * x[ds][e], eq);
      split8(x[ds], qh[ds], ql[ds]);
    }
  }

  v16f o[NB];
#pragma unroll
  for (int d = 0; d < NB; d++)
#pragma unroll
    for (int r = 0; r < 16; r++) o[d][r] = 0.f;
  keep(o);
  float m = -3.402823466e38f, l = 0.f;  // finite: a difference of two is no NaN
  if constexpr (STORED) {
    // Read as constants, through the scalar cache: a vector load in the loop would wait
    // for the stages on their way.
    const auto *uniform = (const __attribute__((address_space(4))) float *)scales;
    for (int st = st0; st < (odd ? st0 : st1); st++) {
      wait_vm_le<FPW, NS - 2>(min(NS - 2, st1 - 1 - st));
      block_barrier();
      if (st + NS - 1 < st1) fetch(st + NS - 1);
      if (kStageKeys * st > wend) continue;  // nothing here is seen by this wave
      const float kinv = uniform[4 * st], vinv = uniform[4 * st + 1];
      const int er = vinv > 0.f ? (__float_as_int(vinv) >> 23) - 127 - unit : 0;
      stage<NB, false>((const h8 *)ring[(st - st0) % NS] + lane, qh, ql, qf * kinv, kStageKeys * st, my, all,
                   h, er, o, m, l, [](int) {}, [] {});
    }
  } else if (st0 < st1) {
    // While a stage is used the next one is made, between the products, and the one
    // behind that is loaded: one barrier a stage.
    post(0);
    lds_barrier();
    uint2 top = tops(0);
    int first = -1000;  // O's first scaling
#pragma unroll
    for (int i = 0; i < 2 * NB; i++) make(ring[0], top, i);
    key_tops(0);
    if (st0 + 1 < st1) {
      load(st0 + 1);
      post(1);
    }
    for (int st = st0, slot = 0; st < st1; st++) {
      const int at = (st - st0) & 1, slot1 = slot == 2 ? 0 : slot + 1, slot2 = slot1 == 2 ? 0 : slot1 + 1;
      lds_barrier();  // this stage and the sizes of the next are there, the last one's slot is free
      const uint2 next = tops(at ^ 1);
      const uint32_t kt = top.x, vt = top.y;
      odd |= max(kt, vt) >= 0x7f800000u;
      {  // far below the largest, and not 0; V is scaled to 2^14, and 0x3c00 is f16's 1
        const uint32_t x = key_s[slot][0][r32], y = key_s[slot][1][r32];
        bool low = (x && x + (kSpread << 23) < kt) || (y && y < 0x3c00u);
        if (vt && __any(y == 0)) {  // zeros, or what f16 has no number for
          const float *v = vp + (int64_t)min(kStageKeys * st + r32, z.nk - 1) * a.v_row;
          for (int d = 0; y == 0 && !low && d < a.hs; d++) low = v[d] != 0.f;
        }
        odd |= __any(low);
      }
      const int e = vt ? -lift(vt) : unit;  // a stage of zeros has no size
      keep(o);
      if (e > unit) {
        if (unit > -1000) {
          const float down = ldexpf(1.f, unit - e);
#pragma unroll
          for (int d = 0; d < NB; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[d][r] *= down;
          keep(o);
        }
        keep(o);
        unit = e;
      }
      keep(o);
      if (first == -1000) first = unit;
      const int er = e - unit;  // (-1000 less itself where V has been 0 so far)
      odd |= er < -kSpread || unit - first > kClimb;
      // (waves that see nothing of the stage have weights of 0; behind the last stage it is made again)
      stage<NB, true>((const h8 *)ring[at] + lane, qh, ql, qf * power(-lift(kt)), kStageKeys * st, my, all, h,
                    max(er, -kSpread), o, m, l, [&](int i) { make(ring[at ^ 1], next, i); },
                    [&] {
                      key_tops(slot1);
                      if (threadIdx.x < 32) key_s[slot2][1][r32] = 0;  // for the stage behind the next
                      if (st + 2 < st1) load(st + 2);
                    });
      if (st + 2 < st1) post(at);
      top = next;
      slot = slot1;
    }
  }
  const int64_t part_row = ((int64_t)split * a.tq + z.qb) * (args.hk * a.group) + un.head;
  const int part_step = args.hk * a.group;
  if (odd || wide) {
    // In fp32, the wave's 32 queries 16 at a time over the block's keys.
    for (int q0 = row0; !idle && q0 < min(row0 + 32, z.nq); q0 += 16) {
      const int r16 = lane & 15, g = lane >> 4, r = min(q0 + r16, z.nq - 1);
      v4f y[2 * NB];
      attend16<2 * NB, VEC>(a, a.q + (int64_t)(z.qb + r) * a.q_row + un.head * a.q_head, kp, vp, r + off,
                            q0 + off, min(min(q0 + 15, z.nq - 1) + off, kStageKeys * st1 - 1),
                            kStageKeys * st0, 16, y, m, l);
      if (q0 + r16 >= z.nq) continue;
      const int64_t at = part_row + (int64_t)r * part_step;
      float *out = args.splits > 1 ? args.part + at * a.hs
                                   : a.out + (int64_t)(z.qb + r) * a.o_row + un.head * a.o_head;
      if (args.splits > 1 && g == 0) args.stat[at] = make_float2(m * 1.44269504f, l);
      const float f = args.splits == 1 && r + off < 0 ? 0.f : one_over(l, args.splits);
#pragma unroll
      for (int j = 0; j < 2 * NB; j++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (16 * j + 4 * g + e < a.hs) out[16 * j + 4 * g + e] = y[j][e] * f;
    }
    return;
  }
  if (idle || row0 + r32 >= z.nq) return;
  {
    float u = l, v = l;
    permlane32_swap(u, v);
    l = u + v;
  }
  // Two factors: the scaling, exact, and 1 / l.  One number for both would lose bits to
  // gradual underflow where V is tiny.
  const float scale = unit > -1000 ? ldexpf(1.f, unit - 13) : 0.f;
  const bool none = args.splits == 1 && my < 0;
  const float f = one_over(l, args.splits);
  float *out;
  if (args.splits > 1) {
    const int64_t at = part_row + (int64_t)row * part_step;
    out = args.part + at * a.hs;
    if (h == 0) args.stat[at] = make_float2(m, l);
  } else {
    out = a.out + (int64_t)(z.qb + row) * a.o_row + un.head * a.o_head;
  }
#pragma unroll
  for (int d = 0; d < NB; d++)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int at = 32 * d + 2 * r + 4 * h;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = none ? 0.f : o[d][r + e] * f * scale;
      if (VEC) {
        if (at < a.hs) *(float4 *)(out + at) = make_float4(y[0], y[1], y[2], y[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (at + e < a.hs) out[at + e] = y[e];
      }
    }
}

// 1024 values of one row, heads side by side: their splits together, four to a thread.
// 273 rows of 32 heads of 100 in up to 9 pieces: 9.5 us for 26 MB, 2.8 TB/s.
template <bool VEC>
__global__ void __launch_bounds__(256) attn_join_k(const F16Args args) {
  extern __shared__ float weight[];  // [heads of the block, ns]
  const PackedArgs &a = args.p;
  const int heads = args.hk * a.group, row = blockIdx.x, tid = threadIdx.x;
  const int s = last_of(a.n, [&](int i) { return clampi(a.q_starts[i], 0, a.tq) <= row; });
  const Seq z = seq_of(a, s);
  if (row < z.qb || row >= z.qb + z.nq) return;
  const int last = row - z.qb + z.nk - z.nq;  // the row's last key
  const int ns = last < 0 ? 0 : last / kStageKeys / args.chunk + 1;
  const int64_t step = (int64_t)a.tq * heads;
  const int e0 = 1024 * (int)blockIdx.y, h0 = e0 / a.hs, h1 = min(heads, (e0 + 1023) / a.hs + 1);
  for (int t = tid; h0 + t < h1; t += 256) {
    const float2 *stat = args.stat + (int64_t)row * heads + h0 + t;
    float M = -INFINITY, L = 0.f;
#pragma unroll 8
    for (int i = 0; i < ns; i++) M = fmaxf(M, stat[i * step].x);
    if (M == -INFINITY) M = 0.f;  // every score is -inf: the sums are 0 too, and the row 0 / 0
#pragma unroll 8
    for (int i = 0; i < ns; i++) {
      const float2 ml = stat[i * step];
      const float f = pow2(ml.x - M) * ml.y;
      weight[t * ns + i] = f;
      L += f;
    }
    for (int i = 0; i < ns; i++) weight[t * ns + i] /= L;
  }
  __syncthreads();
  const float *part = args.part + (int64_t)row * heads * a.hs;
  float *out = a.out + row * a.o_row;
  if (VEC) {
    const int e = e0 + 4 * tid, h = e / a.hs;
    if (h >= heads) return;
    const float *w = weight + (h - h0) * ns;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int i = 0; i < ns; i++) {
      const float4 x = *(const float4 *)(part + i * step * a.hs + e);
      o.x = fmaf(w[i], x.x, o.x);
      o.y = fmaf(w[i], x.y, o.y);
      o.z = fmaf(w[i], x.z, o.z);
      o.w = fmaf(w[i], x.w, o.w);
    }
    *(float4 *)(out + h * a.o_head + (e - h * a.hs)) = o;
  } else {
    for (int e = e0 + tid; e < min(e0 + 1024, heads * a.hs); e += 256) {
      const int h = e / a.hs;
      float o = 0.f;
#pragma unroll 8
      for (int i = 0; i < ns; i++) o = fmaf(weight[(h - h0) * ns + i], part[i * step * a.hs + e], o);
      out[h * a.o_head + (e - h * a.hs)] = o;
    }
  }
}

template <int NB, int NW, int NS, bool VEC, bool STORED>
void launch_f16(const F16Args &a, hipStream_t st) {
  const int heads = a.hk * a.p.group;
  if (STORED)
    hipLaunchKernelGGL((attn_stages_k<NB, VEC>), dim3((unsigned)a.slots, (unsigned)a.hk), dim3(256), 0, st, a);
  hipLaunchKernelGGL((attn_f16_k<NB, NW, NS, VEC, STORED>), dim3((unsigned)(a.blocks * a.hk), (unsigned)a.splits),
                     dim3(64 * NW), 0, st, a);
  if (a.splits > 1)
    hipLaunchKernelGGL(attn_join_k<VEC>, dim3((unsigned)a.p.tq, (unsigned)cdiv((int64_t)heads * a.p.hs, 1024)),
                       dim3(256), (unsigned)(4 * a.splits * std::min<int64_t>(heads, 1024 / a.p.hs + 2)), st, a);
}

// How a call is computed, and where in its scratch what lies.
struct Plan {
  F16Args a;
  int nb;
  bool stored;
  size_t frags, scales, part, stat, bytes;  // offsets, and all of it
};

int plan_packed(const PackedArgs &p, int heads, bool may_store, Plan &plan) {
  plan.nb = p.hs <= 32 ? 1 : p.hs <= 64 ? 2 : p.hs <= 96 ? 3 : p.hs <= 128 ? 4 : p.hs <= 192 ? 6 : 8;
  F16Args &a = plan.a = F16Args{};
  a.p = p;
  a.hk = heads / p.group;
  // attn_stages_k and its traffic pay where about 24 blocks of four waves or more would
  // make each stage: 1024 tokens of 32 heads over 8, 128 wide (32 blocks) 63 us against 77,
  // 4096 (128) 400 against 537; 512 (16) 46 against 39, 2048 of 16 over 16, 64 wide (16) 75
  // against 66.
  // Lengths are on the device, so this and the split below go by the mean.  Batches of like
  // sequences are what it was measured with; uneven ones pay (4096 tokens and 31 single ones
  // beside them 499 us, alone 400; 64 single queries, one of them after 60000 tokens, 4.2 ms).
  const int64_t rows = cdiv(p.tq, p.n), keys = cdiv(p.tk, p.n);
  const bool stored = plan.stored = may_store && rows * p.group >= 24 * 128;
  // Eight waves share a fetched stage where their registers leave room for two on a SIMD.
  const int nw = stored && p.hs <= 128 ? 8 : 4;
  const int64_t slots = p.tk / kStageKeys + p.n, blocks = (int64_t)(p.tq / 32 + p.n) * p.group / nw + p.n;
  if (blocks > UINT32_MAX / a.hk / (64 * nw) || slots > UINT32_MAX / 256)
    return set_error(SIMP_RT_EUNSUPPORTED, "attention_packed: more rows, heads or sequences than the grid holds");
  a.slots = (int)slots;
  a.blocks = (int)blocks;
  // The keys are split where the blocks (each with about `stages`, the last one of a row
  // half used) would not fill the chip, and the rows are long enough to be worth joining:
  // 17 queries after 2983 tokens 28 us against 203, 273 of the 3B heads after up to 1500 56
  // against 126, 2048 tokens of 16 heads 66 against 100.  Shorter pieces than 6 stages cost
  // more in joining than they spare (512 tokens of 32 heads 39 us, 42 with four).
  a.splits = 1;
  a.chunk = INT32_MAX / 2;
  const int64_t cus = num_cus(), room = nw == 8 || p.hs > 128 ? cus : cus * 5 / 2;
  const int64_t wgs = cdiv(cdiv(rows, 32) * p.group, nw) * p.n * a.hk;
  const int64_t stages = cdiv(std::max<int64_t>(keys - rows / 2, 1), kStageKeys);
  if (wgs < room) {
    // One sequence may have all keys.  The pieces' rows take up to 128 MB, and the weights of
    // a block of attn_join_k up to 48 KB.
    const int64_t most = cdiv(p.tk, kStageKeys), row = (int64_t)heads * p.hs;
    const int64_t join_heads = std::min<int64_t>(heads, 1024 / p.hs + 2);
    const int64_t chunk = std::max({int64_t(6), cdiv(cdiv(wgs * stages, room - wgs / 2), 2) * 2,
                                    cdiv(most * join_heads, 12288), cdiv(most * p.tq * row, int64_t(1) << 25)});
    if (cdiv(keys, kStageKeys) >= 2 * chunk) {
      a.chunk = (int)chunk;
      a.splits = (int)cdiv(most, chunk);
    }
  }
  const size_t parts = a.splits > 1 ? (size_t)a.splits * p.tq * heads : 0;
  plan.bytes = 0;
  auto take = [&](size_t n) { return std::exchange(plan.bytes, plan.bytes + (n + 15) / 16 * 16); };
  plan.frags = take(stored ? (size_t)a.slots * a.hk * plan.nb * 8 * 1024 : 0);
  plan.scales = take(stored ? (size_t)a.slots * a.hk * sizeof(float4) : 0);
  plan.part = take(parts * p.hs * 4);
  plan.stat = take(parts * sizeof(float2));
  return SIMP_RT_OK;
}

int launch_packed(const PackedArgs &p, int heads, bool vec, hipStream_t st) {
  Plan plan;
  int rc = plan_packed(p, heads, true, plan);
  if (rc) return rc;
  Workspace ws;
  char *w = nullptr;
  // The stages take as much memory as K and V.  Where there is none, or a captured call's
  // warm-up left none, the blocks make them for themselves.
  if (plan.stored && !ws.try_get(st, plan.bytes, (void **)&w, 9) &&
      (rc = plan_packed(p, heads, false, plan)))
    return rc;
  if (!plan.stored && plan.bytes && (rc = ws.get(st, plan.bytes, (void **)&w, 9))) return rc;
  F16Args &a = plan.a;
  if (w) {
    a.frags = (uint4 *)(w + plan.frags);
    a.scales = (float4 *)(w + plan.scales);
    a.part = (float *)(w + plan.part);
    a.stat = (float2 *)(w + plan.stat);
  }
#define F16(NB, NW, NS, STORED) \
  vec ? launch_f16<NB, NW, NS, true, STORED>(a, st) : launch_f16<NB, NW, NS, false, STORED>(a, st)
  if (plan.stored) {
    switch (plan.nb) {
      case 1: F16(1, 8, 4, true); break;
      case 2: F16(2, 8, 4, true); break;
      case 3: F16(3, 8, 4, true); break;
      case 4: F16(4, 8, 4, true); break;
      case 6: F16(6, 4, 3, true); break;
      default: F16(8, 4, 2, true);
    }
  } else {
    switch (plan.nb) {
      case 1: F16(1, 4, 2, false); break;
      case 2: F16(2, 4, 2, false); break;
      case 3: F16(3, 4, 2, false); break;
      case 4: F16(4, 4, 2, false); break;
      case 6: F16(6, 4, 2, false); break;
      default: F16(8, 4, 2, false);
    }
  }
#undef F16
  return SIMP_RT_OK;
}

}  // namespace
}  // namespace simp

using namespace simp;

extern "C" {

int32_t simp_rt_attention_packed_f32(
    const float *q_alloc, const float *q, int64_t q_off, int64_t q_s0, int64_t q_s1, int64_t q_s2,
    int64_t q_st0, int64_t q_st1, int64_t q_st2, const float *k_alloc, const float *k,
    int64_t k_off, int64_t k_s0, int64_t k_s1, int64_t k_s2, int64_t k_st0, int64_t k_st1,
    int64_t k_st2, const float *v_alloc, const float *v, int64_t v_off, int64_t v_s0, int64_t v_s1,
    int64_t v_s2, int64_t v_st0, int64_t v_st1, int64_t v_st2, float *out_alloc, float *out,
    int64_t out_off, int64_t out_s0, int64_t out_s1, int64_t out_s2, int64_t out_st0,
    int64_t out_st1, int64_t out_st2, const int32_t *qst_alloc, const int32_t *q_starts,
    int64_t qst_off, int64_t qst_size, int64_t qst_stride, const int32_t *kst_alloc,
    const int32_t *k_starts, int64_t kst_off, int64_t kst_size, int64_t kst_stride, double scale) {
  (void)q_alloc; (void)k_alloc; (void)v_alloc; (void)out_alloc; (void)qst_alloc; (void)kst_alloc;
  int rc;
  Desc3<const float> dq{q, q_off, {q_s0, q_s1, q_s2}, {q_st0, q_st1, q_st2}, 0};
  Desc3<const float> dk{k, k_off, {k_s0, k_s1, k_s2}, {k_st0, k_st1, k_st2}, 0};
  Desc3<const float> dv{v, v_off, {v_s0, v_s1, v_s2}, {v_st0, v_st1, v_st2}, 0};
  Desc3<float> dout{out, out_off, {out_s0, out_s1, out_s2}, {out_st0, out_st1, out_st2}, 0};
  if ((rc = dq.check("q")) || (rc = dk.check("k")) || (rc = dv.check("v")) ||
      (rc = dout.check("out")) || (rc = check_desc1("q_starts", q_starts, qst_off, qst_size, qst_stride)) ||
      (rc = check_desc1("k_starts", k_starts, kst_off, kst_size, kst_stride)))
    return rc;
  if (!dout.is(q_s0, q_s1, q_s2) || !dv.is(k_s0, k_s1, k_s2) || k_s2 != q_s2)
    return set_error(SIMP_RT_EINVAL, "attention_packed: shape mismatch: q and out [%lld,%lld,%lld], "
                     "k and v [%lld,%lld,%lld]", (long long)q_s0, (long long)q_s1, (long long)q_s2,
                     (long long)k_s0, (long long)k_s1, (long long)k_s2);
  if (qst_size < 1 || kst_size != qst_size)
    return set_error(SIMP_RT_EINVAL, "attention_packed: q_starts and k_starts must have sequences + 1 entries");
  if (!scale_fits(scale))
    return set_error(SIMP_RT_EINVAL, "attention_packed: scale must be finite, also in fp32 and times log2(e)");
  if (q_s2 < 1 || q_s2 > 256)
    return set_error(SIMP_RT_EUNSUPPORTED, "attention_packed: head_size %lld is not in 1..256", (long long)q_s2);
  if (k_s1 < 1 || q_s1 % k_s1 != 0)
    return set_error(SIMP_RT_EINVAL, "attention_packed: %lld heads are no multiple of %lld kv heads",
                     (long long)q_s1, (long long)k_s1);
  const int64_t n = qst_size - 1;
  if (q_s0 == 0 || q_s1 == 0 || n == 0) return SIMP_RT_OK;
  if (q_s0 > INT32_MAX - 64 || k_s0 > INT32_MAX - 64 || q_s1 > 65535 || n > INT32_MAX / 65536)
    return set_error(SIMP_RT_EUNSUPPORTED, "attention_packed: more rows, heads or sequences than the grid holds");
  if (dk.st[0] >= 1 << 23 || dv.st[0] >= 1 << 23)  // 32-bit offsets within 32 rows
    return set_error(SIMP_RT_EUNSUPPORTED, "attention_packed: rows of k or v 2^23 elements or more apart");
  if (overlap(dout.data(), dout.bytes(), dq.data(), dq.bytes()) ||
      overlap(dout.data(), dout.bytes(), dk.data(), dk.bytes()) ||
      overlap(dout.data(), dout.bytes(), dv.data(), dv.bytes()) ||
      overlap(dout.data(), dout.bytes(), q_starts + qst_off, 4 * (size_t)qst_size) ||
      overlap(dout.data(), dout.bytes(), k_starts + kst_off, 4 * (size_t)kst_size))
    return set_error(SIMP_RT_EINVAL, "attention_packed: out shares memory with an input");
  const int dev = ensure_device();
  if (dev < 0) return dev;
  Operand oq, ok, ov, oo, oqs, oks;
  if ((rc = bind_here(oq, dq.data(), dq.bytes(), Operand::kIn, dev, "q")) ||
      (rc = bind_here(ok, dk.data(), dk.bytes(), Operand::kIn, dev, "k")) ||
      (rc = bind_here(ov, dv.data(), dv.bytes(), Operand::kIn, dev, "v")) ||
      (rc = bind_here(oo, dout.data(), dout.bytes(), Operand::kOut, dev, "out")) ||
      (rc = bind_here(oqs, q_starts + qst_off, 4 * (size_t)qst_size, Operand::kIn, dev, "q_starts")) ||
      (rc = bind_here(oks, k_starts + kst_off, 4 * (size_t)kst_size, Operand::kIn, dev, "k_starts")))
    return rc;
  PackedArgs a;
  a.q = (const float *)oq.dev();
  a.k = (const float *)ok.dev();
  a.v = (const float *)ov.dev();
  a.out = (float *)oo.dev();
  a.q_starts = (const int *)oqs.dev();
  a.k_starts = (const int *)oks.dev();
  a.q_row = dq.st[0], a.q_head = dq.st[1], a.k_row = dk.st[0], a.k_head = dk.st[1];
  a.v_row = dv.st[0], a.v_head = dv.st[1], a.o_row = dout.st[0], a.o_head = dout.st[1];
  a.tq = (int)q_s0, a.tk = (int)k_s0, a.n = (int)n;
  a.group = (int)(q_s1 / k_s1), a.hs = (int)q_s2;
  a.scale = (float)scale;
  const bool vec = a.hs % 4 == 0 &&
                   ((a.q_row | a.q_head | a.k_row | a.k_head | a.v_row | a.v_head | a.o_row | a.o_head) & 3) == 0 &&
                   (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) & 15) == 0;
  if ((rc = launch_packed(a, (int)q_s1, vec, cur_stream()))) return rc;
  Operand *ops[] = {&oq, &ok, &ov, &oo, &oqs, &oks};
  return finish(ops, 6);
}

}  // extern "C"
