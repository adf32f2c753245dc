// attention.hip -- causal attention of packed prompts (simp_rt_attention_packed_f32).
//
// out_i = sum_j p_ij v_j, p_i = softmax_j(scale q_i . k_j) over the keys j <= i +
// nk - nq of the row's sequence.  One pass over the keys with a running maximum m
// and sum l: o and l are scaled by e^(m_old - m_new) when a tile raises m.
#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <utility>

#include "rt_device.h"
#include "serve_args.h"

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

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return min(max(x, lo), hi); }

// The sequence of tile slot `t`, where sequence s has the slots q_starts[s] / R + s
// and on: R rows a tile, so at most n_q / R + 1 of them, and the next one's begin
// behind.  Ends with 0 <= s < n whatever the starts hold.
template <int R>
__device__ __forceinline__ int seq_of_slot(const int *starts, int n, int rows, int t) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (clampi(starts[mid], 0, rows) / R + mid <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
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

template <int HB>
struct TileLds {
  float o[4][16 * HB][17];
  float m[4][16], l[4][16];
};

// A block takes 16 queries of one head (tile slot t); its four waves take the 16-key
// tiles in turn, each with its own running maximum, sum and output, combined through LDS
// at the end.  only: sequences to take part (n of them, kv heads apart), or null.
template <int HB, bool VEC>
__device__ __forceinline__ void f32_tile(const PackedArgs &a, int t, int h, const int *only,
                                         TileLds<HB> &lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r16 = lane & 15, g = lane >> 4, hs = a.hs;
  const int s = seq_of_slot<16>(a.q_starts, a.n, a.tq, t);
  const int qb = clampi(a.q_starts[s], 0, a.tq), qe = clampi(a.q_starts[s + 1], qb, a.tq);
  const int kb = clampi(a.k_starts[s], 0, a.tk), ke = clampi(a.k_starts[s + 1], kb, a.tk);
  const int nq = qe - qb, nk = ke - kb;
  const int slot0 = qb / 16 + s;
  if (t < slot0 || t - slot0 >= (nq + 15) / 16) return;
  if (only && !only[(int64_t)(h / a.group) * a.n + s]) return;
  const int q0 = 16 * (t - slot0), row = min(q0 + r16, nq - 1);
  v4f o[HB];
  float m, l;
  attend16<HB, VEC>(a, a.q + (int64_t)(qb + row) * a.q_row + h * a.q_head,
                    a.k + (int64_t)kb * a.k_row + (h / a.group) * a.k_head,
                    a.v + (int64_t)kb * a.v_row + (h / a.group) * a.v_head, row + nk - nq,
                    q0 + nk - nq, min(q0 + 15, nq - 1) + nk - nq, 16 * wave, 64, o, m, l);
  if (g == 0) {
    lds.m[wave][r16] = m;
    lds.l[wave][r16] = l;
  }
#pragma unroll
  for (int j = 0; j < HB; j++)
#pragma unroll
    for (int r = 0; r < 4; r++) lds.o[wave][16 * j + 4 * g + r][r16] = o[j][r];
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * hs; e += 256) {
    const int qi = e / hs, d = e - qi * hs;
    if (q0 + qi >= nq) break;  // queries in increasing order
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) M = fmaxf(M, lds.m[w][qi]);
    const float mu = M == -INFINITY ? 0.f : M;
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float f = expf(lds.m[w][qi] - mu);
      num = fmaf(f, lds.o[w][d][qi], num);
      den = fmaf(f, lds.l[w][qi], den);
    }
    const bool none = q0 + qi + nk - nq < 0;
    a.out[(int64_t)(qb + q0 + qi) * a.o_row + h * a.o_head + d] = none ? 0.f : num / den;
  }
}

template <int HB, bool VEC>
__global__ void __launch_bounds__(256) attn_f32_k(const PackedArgs a) {
  __shared__ TileLds<HB> lds;
  f32_tile<HB, VEC>(a, (int)(gridDim.x - 1 - blockIdx.x), blockIdx.y, nullptr, lds);
}

// ---- the split form
//
// Longer inputs run both products on v_mfma_f32_32x32x16_f16.  A number x, scaled by
// a power of two to below 2^15, is hi + lo + r with hi = f16(x), lo = f16(x - hi) and
// |r| <= 2^-22 |x| (2^-40 of the scaling's unit for the smallest); x y is taken as
// hi hi + hi lo + lo hi, each product exact and each sum fp32.  That is as close as
// an fp32 product, at three times an f16 product's cost instead of the fp32 matrix
// instruction's sixteen.
//   attn_split_k  takes K and V apart once: per 32 keys of a kv head a stage of
//                 1 KB operand fragments in the order that the matrix instruction's
//                 lanes want them, so that attn_f16_k moves them to LDS as they
//                 are; and the two scalings (NaN where a value is not finite).
//   attn_f16_k    a block of NW waves takes NW units (32 queries of one head) of one kv
//                 head, so that the query heads of a group share the fragments, and
//                 walks the stages through a ring in LDS.  S^T = K Q^T leaves a lane
//                 with 16 keys of one query, which are the B operand of O^T +=
//                 V^T P^T in the order that attn_split_k laid the keys of V.
//   attn_join_k   where there are few units the keys are split over several blocks; this
//                 joins what they leave.
//   attn_again_k  computes the sequences in fp32 whose keys the split form does not serve.

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));

#ifndef AHEAD
#define AHEAD 4
#endif
constexpr int kStageKeys = 32;
// Where keys differ in size by more than this, the smaller ones' parts lie too low in
// the larger ones' scaling (they keep at least 24 bits up to here), and a key that a
// query does not see would cost the row bits: those rows are computed in fp32.
constexpr float kSpread = 1.f / 16384;

struct SplitArgs {
  PackedArgs p;
  uint4 *frags;    // [slots, kv heads] stages
  float4 *scales;  // [kv heads, slots]: 1 / the scaling of K, of V, and the smallest key's
  int *any;        // whether some sequence goes to attn_again_k
  int *again;      // [kv heads, n]: which
  int hk, slots;
};

// 2^x, below 2^-126 as 0
__device__ __forceinline__ float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// The exponent that brings a largest magnitude into [2^14, 2^15)
__device__ __forceinline__ int lift(float top) {
  const int e = top > 0.f ? 14 - ilogbf(top) : 0;
  return min(e, 126);
}

__device__ __forceinline__ void split8(const float (&x)[8], h8 &hi, h8 &lo) {
  typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const h2 h = __builtin_convertvector((f2{x[e], x[e + 1]}), h2);
    const f2 r = {fmaf((float)h[0], -1.f, x[e]), fmaf((float)h[1], -1.f, x[e + 1])};
    const h2 l = __builtin_convertvector(r, h2);
    hi[e] = h[0], hi[e + 1] = h[1];
    lo[e] = l[0], lo[e + 1] = l[1];
  }
}

// One stage.  NB: 32-dimension blocks of a head.
template <int NB, bool VEC>
__global__ void __launch_bounds__(256) attn_split_k(const SplitArgs a) {
  constexpr int DP = 32 * NB, LD = DP + 4;
  __shared__ float tile[2][32][LD];
  __shared__ float most[4], least[4];
  const PackedArgs &p = a.p;
  const int slot = blockIdx.x, hk = blockIdx.y, tid = threadIdx.x;
  if (slot == 0 && hk == 0 && tid == 0) *a.any = 0;
  const int s = seq_of_slot<kStageKeys>(p.k_starts, p.n, p.tk, slot);
  const int kb = clampi(p.k_starts[s], 0, p.tk), ke = clampi(p.k_starts[s + 1], kb, p.tk);
  const int slot0 = kb / kStageKeys + s;
  if (slot < slot0) return;
  const int64_t key0 = (int64_t)(slot - slot0) * kStageKeys;
  if (key0 >= ke - kb) return;
  const int nk = (int)min((int64_t)kStageKeys, ke - kb - key0);
  bool odd = false;
#pragma unroll
  for (int w = 0; w < 2; w++) {
    const float *x = w ? p.v + (kb + key0) * p.v_row + hk * p.v_head
                       : p.k + (kb + key0) * p.k_row + hk * p.k_head;
    const int64_t row = w ? p.v_row : p.k_row;
    for (int e = tid; e < 32 * DP / 4; e += 256) {
      const int r = e / (DP / 4), d = 4 * (e - r * (DP / 4));
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < nk) v = load4<VEC>(x + r * row, d, p.hs);
      *(float4 *)&tile[w][r][d] = v;
      odd |= !(fabsf(v.x) < INFINITY && fabsf(v.y) < INFINITY && fabsf(v.z) < INFINITY &&
               fabsf(v.w) < INFINITY);
    }
  }
  const bool bad = __syncthreads_or(odd);
  {  // the largest of each key, four threads to one
    const int w = tid >> 7, r = (tid >> 2) & 31, c = tid & 3;
    float t = 0.f;
    for (int d = 4 * c; d < DP; d += 16) {
      const float4 v = *(const float4 *)&tile[w][r][d];
      t = fmaxf(t, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
    }
    t = fmaxf(t, __shfl_xor(t, 1));
    t = fmaxf(t, __shfl_xor(t, 2));
    float lowest = t > 0.f ? t : INFINITY;
    t = wave_max(t);
    lowest = -wave_max(-lowest);
    if ((tid & 63) == 0) {
      most[tid >> 6] = t;
      least[tid >> 6] = lowest;
    }
  }
  __syncthreads();
  const float kt = fmaxf(most[0], most[1]), vt = fmaxf(most[2], most[3]);
  const float kl = fminf(least[0], least[1]), vl = fminf(least[2], least[3]);
  const int ek = lift(kt), ev = lift(vt);
  if (tid == 0) {
    const bool wide = bad || kl < kt * kSpread;
    a.scales[(int64_t)hk * a.slots + slot] =
        make_float4(ldexpf(1.f, -ek), wide ? NAN : vt > 0.f ? ldexpf(1.f, -ev) : 0.f, vl, 0.f);
  }
  if (bad) return;
  uint4 *out = a.frags + ((int64_t)slot * a.hk + hk) * (NB * 8 * 64);
  const int lane = tid & 63, r32 = lane & 31, h = lane >> 5;
  for (int f = tid >> 6; f < 2 * NB; f += 4) {  // K: 16 dimensions, 32 keys
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = ldexpf(tile[0][r32][16 * f + 8 * h + e], ek);
    h8 hi, lo;
    split8(x, hi, lo);
    out[(2 * f) * 64 + lane] = __builtin_bit_cast(uint4, hi);
    out[(2 * f + 1) * 64 + lane] = __builtin_bit_cast(uint4, lo);
  }
  for (int f = tid >> 6; f < 2 * NB; f += 4) {  // V: 16 keys (f / NB), 32 dimensions
    const int i = f / NB, db = f - i * NB;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++)
      x[e] = ldexpf(tile[1][16 * i + 8 * (e >> 2) + 4 * h + (e & 3)][32 * db + r32], ev);
    h8 hi, lo;
    split8(x, hi, lo);
    out[(4 * NB + 2 * f) * 64 + lane] = __builtin_bit_cast(uint4, hi);
    out[(4 * NB + 2 * f + 1) * 64 + lane] = __builtin_bit_cast(uint4, lo);
  }
}

struct F16Args {
  SplitArgs s;
  int blocks;   // of one kv head and one split
  int splits, chunk;  // of the keys: stages a split takes
  float *part;  // [splits, tq, heads, head_size], scaled by the row's sum; with splits
  float2 *stat; // [splits, tq, heads]
};

// NB: 32-dimension blocks; NW: waves; NS: stages in the ring.
template <int NB, int NW, int NS, bool VEC>
__global__ void __launch_bounds__(64 * NW) attn_f16_k(const F16Args args) {
  constexpr int kFrags = 8 * NB, FPW = kFrags / NW;  // fragments of a stage; loaded by a wave
  static_assert(kFrags % NW == 0, "each wave loads as many fragments");
  __shared__ uint4 ring[NS][kFrags * 64];
  __shared__ float vtop_s[NW], vlow_s[NW];
  const SplitArgs &sa = args.s;
  const PackedArgs &a = sa.p;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r32 = lane & 31, h = lane >> 5;
  // the last rows of a sequence, which see most keys, come first
  const int hk = blockIdx.x % sa.hk, split = blockIdx.y;
  const int w = args.blocks - 1 - blockIdx.x / sa.hk;
  // Sequence s has the blocks ((q_starts[s] / 32 + s) G / NW) + s and on.
  const int G = a.group;
  auto base = [&](int s) {
    return (int)(((int64_t)(clampi(a.q_starts[s], 0, a.tq) / 32 + s) * G) / NW) + s;
  };
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (base(mid) <= w) lo = mid;
    else hi = mid - 1;
  }
  const int seq = lo, b0 = base(seq);
  const int qb = clampi(a.q_starts[seq], 0, a.tq), qe = clampi(a.q_starts[seq + 1], qb, a.tq);
  const int kb = clampi(a.k_starts[seq], 0, a.tk), ke = clampi(a.k_starts[seq + 1], kb, a.tk);
  const int nq = qe - qb, nk = ke - kb, tiles = (nq + 31) / 32;
  if (w < b0 || (int64_t)(w - b0) * NW >= (int64_t)tiles * G) return;
  const int64_t unit = (int64_t)(w - b0) * NW + wave;
  const int tile = (int)(unit / G), head = hk * G + (int)(unit - (int64_t)tile * G);
  const bool idle = tile >= tiles;
  const int row0 = 32 * tile, row = min(row0 + r32, nq - 1);  // this lane's query
  const int my = row + nk - nq;                               // its last key, or negative
  const int first = row0 + nk - nq;                           // what every query sees, at least
  const int wend = idle ? -1 : min(row0 + 31, nq - 1) + nk - nq;  // the wave's last key
  const int top_tile = min(tiles - 1, (int)(((int64_t)(w - b0) * NW + NW - 1) / G));
  const int bend = min(32 * top_tile + 31, nq - 1) + nk - nq;     // the block's
  const int st0 = split * args.chunk;
  const int st1 = min(bend < 0 ? 0 : bend / kStageKeys + 1, st0 + args.chunk);
  if (split > 0 && st0 >= st1) return;  // attn_join_k does not read it
  const int slot0 = kb / kStageKeys + seq;

  // The largest scaling of V in the block's stages is the unit of O.
  const float4 *scales = sa.scales + (int64_t)hk * sa.slots + slot0;
  float vt = 0.f, vl = INFINITY;
  bool odd = false;
  for (int i = threadIdx.x; i < (nk + kStageKeys - 1) / kStageKeys; i += 64 * NW) {
    const float4 v = scales[i];
    odd |= v.y != v.y;
    vt = fmaxf(vt, v.y);
    vl = fminf(vl, v.z);
  }
  vt = wave_max(vt);
  vl = -wave_max(-vl);
  if (lane == 0) {
    vtop_s[wave] = vt;
    vlow_s[wave] = vl;
  }
  odd = __syncthreads_or(odd);
#pragma unroll
  for (int i = 0; i < NW; i++) {
    vt = fmaxf(vt, vtop_s[i]);
    vl = fminf(vl, vlow_s[i]);
  }
  odd |= vl < vt * (32768.f * kSpread);  // the largest value is below 2^15 vt
  if (split == 0 && threadIdx.x == 0) {
    sa.again[(int64_t)hk * a.n + seq] = odd;  // the same from each of its blocks
    if (odd) *sa.any = 1;
  }
  if (odd) return;

  const uint32_t lds0 = lds_offset(&ring[0][0]);
  auto fetch = [&](int st) {
    const uint4 *src = sa.frags + ((int64_t)(slot0 + st) * sa.hk + hk) * (kFrags * 64) + lane;
    const uint32_t dst = lds0 + (uint32_t)((st - st0) % NS) * (kFrags * 1024);
#pragma unroll
    for (int i = 0; i < FPW; i++) {
      const int f = wave + i * NW;
      dma16(src + f * 64, dst + f * 1024);
    }
  };
#pragma unroll
  for (int i = 0; i < NS - 1; i++)
    if (st0 + i < st1) fetch(st0 + i);

  h8 qh[2 * NB], ql[2 * NB];
  float qf;
  {
    const float *qr = a.q + (int64_t)(qb + row) * a.q_row + head * a.q_head;
    float top = 0.f;
    float x[2 * NB][8];
#pragma unroll
    for (int ds = 0; ds < 2 * NB; ds++) {
      const int d0 = 16 * ds + 8 * h;
      if (VEC) {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
          if (!idle && d0 + e < a.hs) v = *(const float4 *)(qr + d0 + e);
          x[ds][e] = v.x, x[ds][e + 1] = v.y, x[ds][e + 2] = v.z, x[ds][e + 3] = v.w;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) x[ds][e] = !idle && d0 + e < a.hs ? qr[d0 + e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[ds][e]));
    }
    {
      float u = top, v = top;
      permlane32_swap(u, v);
      top = fmaxf(u, v);
    }
    const int eq = top < INFINITY ? lift(top) : 0;  // infinities and NaN come through
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
  float m = -3.402823466e38f, l = 0.f;  // finite: a difference of two is no NaN
  const int vexp = __float_as_int(vt) >> 23;
  // Read as constants, through the scalar cache: a vector load here would wait for the
  // stages on their way.
  const auto *uniform = (const __attribute__((address_space(4))) float *)scales;
  for (int st = st0; st < st1; st++) {
    wait_vm_le<FPW, NS - 2>(min(NS - 2, st1 - 1 - st));
    block_barrier();
    if (st + NS - 1 < st1) fetch(st + NS - 1);
    if (kStageKeys * st > wend) continue;  // nothing here is seen by this wave
    const float kinv = uniform[4 * st], vinv = uniform[4 * st + 1];
    const h8 *frag = (const h8 *)ring[(st - st0) % NS] + lane;
    v16f s;
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] = 0.f;
    // Two fragments are read ahead of the products that use two others: under the
    // other waves' reads one alone comes later than three products take.
    constexpr int kReads = 0x100, kProducts = 0x008;
    {
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
      __builtin_amdgcn_sched_group_barrier(kReads, AHEAD, 0);
#pragma unroll
      for (int ds = 0; ds < 2 * NB; ds++) {
        __builtin_amdgcn_sched_group_barrier(kProducts, 3, 0);
        __builtin_amdgcn_sched_group_barrier(kReads, 2, 0);
      }
    }
    float f = qf * kinv;
    if (kStageKeys * st + 31 > first) {  // some query does not see all of them
#pragma unroll
      for (int r = 0; r < 16; r++)
        s[r] = kStageKeys * st + 8 * (r >> 2) + 4 * h + (r & 3) <= my ? s[r] * f : -INFINITY;
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
    // The maximum is raised only where a weight would pass 4: weights of 2^13 to the
    // largest one's 1 still fit f16 then.
    if (__any(mt > m + 2.f)) {
      const float mn = fmaxf(m, mt), alpha = pow2(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < NB; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] *= alpha;
    }
    // V's scaling over the unit, a power of two 2^er <= 1
    const int er = vinv > 0.f ? (__float_as_int(vinv) >> 23) - vexp : 0;
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
      __builtin_amdgcn_sched_group_barrier(kReads, AHEAD, 1);
#pragma unroll
      for (int d = 0; d < 2 * NB; d++) {
        __builtin_amdgcn_sched_group_barrier(kProducts, 3, 1);
        __builtin_amdgcn_sched_group_barrier(kReads, 2, 1);
      }
    }
    l = fmaf(pl, __int_as_float((127 - 13 - er) << 23), l);
  }
  if (idle || row0 + r32 >= nq) return;
  {
    float u = l, v = l;
    permlane32_swap(u, v);
    l = u + v;
  }
  const float o_unit = vt * (1.f / 8192.f);
  float *out;
  float f;
  if (args.splits > 1) {
    const int64_t at = ((int64_t)split * a.tq + qb + row) * (sa.hk * G) + head;
    out = args.part + at * a.hs;
    f = o_unit;
    if (h == 0) args.stat[at] = make_float2(m, l);
  } else {
    out = a.out + (int64_t)(qb + row) * a.o_row + head * a.o_head;
    f = my < 0 ? 0.f : o_unit / l;
  }
  const bool none = args.splits == 1 && my < 0;
#pragma unroll
  for (int d = 0; d < NB; d++)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int at = 32 * d + 2 * r + 4 * h;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = none ? 0.f : o[d][r + e] * f;
      if (VEC) {
        if (at < a.hs) *(float4 *)(out + at) = make_float4(y[0], y[1], y[2], y[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (at + e < a.hs) out[at + e] = y[e];
      }
    }
}

// One row of one head: its splits together, four rows to a block.
__global__ void __launch_bounds__(256) attn_join_k(const F16Args args) {
  const PackedArgs &a = args.s.p;
  const int lane = threadIdx.x & 63, heads = args.s.hk * a.group;
  const int64_t e = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), row = e / heads;
  const int head = (int)(e - row * heads);
  if (row >= a.tq) return;
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (clampi(a.q_starts[mid], 0, a.tq) <= row) lo = mid;
    else hi = mid - 1;
  }
  const int qb = clampi(a.q_starts[lo], 0, a.tq), qe = clampi(a.q_starts[lo + 1], qb, a.tq);
  const int kb = clampi(a.k_starts[lo], 0, a.tk), ke = clampi(a.k_starts[lo + 1], kb, a.tk);
  if (row < qb || row >= qe) return;
  const int last = (int)(row - qb) + (ke - kb) - (qe - qb);  // the row's last key
  float *out = a.out + row * a.o_row + head * a.o_head;
  if (last < 0) {
    for (int d = lane; d < a.hs; d += 64) out[d] = 0.f;
    return;
  }
  const int ns = last / (kStageKeys * args.chunk) + 1;
  const int64_t step = (int64_t)a.tq * heads, at = row * heads + head;
  float M = -INFINITY;
  for (int s = 0; s < ns; s++) M = fmaxf(M, args.stat[at + s * step].x);
  const float mu = M == -INFINITY ? 0.f : M;
  float L = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < ns; s++) {
    const float2 ml = args.stat[at + s * step];
    const float f = pow2(ml.x - mu);
    L = fmaf(f, ml.y, L);
    const float *part = args.part + (at + s * step) * a.hs;
#pragma unroll
    for (int c = 0; c < 4; c++)
      if (lane + 64 * c < a.hs) o[c] = fmaf(f, part[lane + 64 * c], o[c]);
  }
#pragma unroll
  for (int c = 0; c < 4; c++)
    if (lane + 64 * c < a.hs) out[lane + 64 * c] = o[c] / L;
}

// The sequences that attn_f16_k left out.
template <int HB, bool VEC>
__global__ void __launch_bounds__(256) attn_again_k(const SplitArgs a, int tiles) {
  __shared__ TileLds<HB> lds;
  if (!*a.any) return;
  const int64_t items = (int64_t)tiles * a.hk * a.p.group;
  for (int64_t e = blockIdx.x; e < items; e += gridDim.x) {
    f32_tile<HB, VEC>(a.p, (int)(e % tiles), (int)(e / tiles), a.again, lds);
    __syncthreads();
  }
}

template <bool VEC>
void launch_f32(const PackedArgs &a, dim3 grid, hipStream_t st) {
#define ATTN(HB) hipLaunchKernelGGL((attn_f32_k<HB, VEC>), grid, dim3(256), 0, st, a)
  if (a.hs <= 32) ATTN(2);
  else if (a.hs <= 64) ATTN(4);
  else if (a.hs <= 128) ATTN(8);
  else ATTN(16);
#undef ATTN
}

template <int NB, int NW, int NS, bool VEC>
void launch_f16_(const F16Args &a, hipStream_t st) {
  const PackedArgs &p = a.s.p;
  hipLaunchKernelGGL((attn_split_k<NB, VEC>), dim3((unsigned)a.s.slots, (unsigned)a.s.hk), dim3(256),
                     0, st, a.s);
  hipLaunchKernelGGL((attn_f16_k<NB, NW, NS, VEC>), dim3((unsigned)(a.blocks * a.s.hk), (unsigned)a.splits),
                     dim3(64 * NW), 0, st, a);
  const int64_t heads = (int64_t)a.s.hk * p.group;
  if (a.splits > 1)
    hipLaunchKernelGGL(attn_join_k, dim3((unsigned)cdiv(p.tq * heads, 4)), dim3(256), 0, st, a);
  const int tiles = p.tq / 16 + p.n;
  hipLaunchKernelGGL((attn_again_k<2 * NB, VEC>), dim3((unsigned)std::min<int64_t>(tiles * heads, 1024)),
                     dim3(256), 0, st, a.s, tiles);
}

// Waves of a block: eight share the fragments where a wave's registers leave room for
// two waves on a SIMD.
int f16_waves(int hs) { return hs <= 128 ? 8 : 4; }

int launch_f16(const PackedArgs &p, int heads, bool vec, hipStream_t st) {
  const int nb = p.hs <= 32 ? 1 : p.hs <= 64 ? 2 : p.hs <= 96 ? 3 : p.hs <= 128 ? 4 : p.hs <= 192 ? 6 : 8;
  const int nw = f16_waves(p.hs);
  F16Args a{};
  a.s.p = p;
  a.s.hk = heads / p.group;
  a.s.slots = p.tk / kStageKeys + p.n;
  a.blocks = (int)((int64_t)(p.tq / 32 + p.n) * p.group / nw) + p.n;
  a.splits = 1;
  a.chunk = INT32_MAX / 2;
  const size_t rows = a.splits > 1 ? (size_t)a.splits * p.tq * heads : 0;
  size_t bytes = 0;
  auto take = [&](size_t n) { return std::exchange(bytes, bytes + (n + 15) / 16 * 16); };
  const size_t frags = take((size_t)a.s.slots * a.s.hk * nb * 8 * 1024);
  const size_t scales = take((size_t)a.s.slots * a.s.hk * sizeof(float4));
  const size_t part = take(rows * p.hs * 4), stat = take(rows * sizeof(float2));
  const size_t any = take(4), again = take((size_t)p.n * a.s.hk * 4);
  Workspace ws;
  char *w;
  if (int rc = ws.get(st, bytes, (void **)&w, 9)) return rc;
  a.s.frags = (uint4 *)(w + frags);
  a.s.scales = (float4 *)(w + scales);
  a.part = (float *)(w + part);
  a.stat = (float2 *)(w + stat);
  a.s.any = (int *)(w + any);
  a.s.again = (int *)(w + again);
#define F16(NB, NW, NS) vec ? launch_f16_<NB, NW, NS, true>(a, st) : launch_f16_<NB, NW, NS, false>(a, st)
  switch (nb) {
    case 1: F16(1, 8, 4); break;
    case 2: F16(2, 8, 4); break;
    case 3: F16(3, 8, 4); break;
    case 4: F16(4, 8, 4); break;
    case 6: F16(6, 4, 3); break;
    default: F16(8, 4, 2);
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
  if (!std::isfinite(scale))
    return set_error(SIMP_RT_EINVAL, "attention_packed: scale must be finite");
  if (q_s2 < 1 || q_s2 > 256)
    return set_error(SIMP_RT_EUNSUPPORTED, "attention_packed: head_size %lld is not in 1..256", (long long)q_s2);
  if (k_s1 < 1 || q_s1 % k_s1 != 0)
    return set_error(SIMP_RT_EINVAL, "attention_packed: %lld heads are no multiple of %lld kv heads",
                     (long long)q_s1, (long long)k_s1);
  const int64_t n = qst_size - 1;
  if (q_s0 == 0 || q_s1 == 0 || n == 0) return SIMP_RT_OK;
  if (q_s0 > INT32_MAX || k_s0 > INT32_MAX || q_s1 > 65535 || n > INT32_MAX - 1 ||
      (q_s0 / 16 + n) * 256 > UINT32_MAX)
    return set_error(SIMP_RT_EUNSUPPORTED, "attention_packed: more rows, heads or sequences than the grid holds");
  if (overlap(dout.data(), dout.bytes(), dq.data(), dq.bytes()) ||
      overlap(dout.data(), dout.bytes(), dk.data(), dk.bytes()) ||
      overlap(dout.data(), dout.bytes(), dv.data(), dv.bytes()))
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
  a.q_row = q_st0, a.q_head = q_st1, a.k_row = k_st0, a.k_head = k_st1;
  a.v_row = v_st0, a.v_head = v_st1, a.o_row = out_st0, a.o_head = out_st1;
  a.tq = (int)q_s0, a.tk = (int)k_s0, a.n = (int)n;
  a.group = (int)(q_s1 / k_s1), a.hs = (int)q_s2;
  a.scale = (float)scale;
  const bool vec = a.hs % 4 == 0 &&
                   ((q_st0 | q_st1 | k_st0 | k_st1 | v_st0 | v_st1 | out_st0 | out_st1) & 3) == 0 &&
                   (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.out) & 15) == 0;
  if (getenv("F16")) {
    if ((rc = launch_f16(a, (int)q_s1, vec, cur_stream()))) return rc;
  } else {
    const dim3 grid((unsigned)(q_s0 / 16 + n), (unsigned)q_s1);
    if (vec) launch_f32<true>(a, grid, cur_stream());
    else launch_f32<false>(a, grid, cur_stream());
  }
  Operand *ops[] = {&oq, &ok, &ov, &oo, &oqs, &oks};
  return finish(ops, 6);
}

}  // extern "C"
