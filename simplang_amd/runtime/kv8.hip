// kv8.hip -- a key/value cache of 8-bit codes with an fp32 scale per block of tokens
// and head: storing rows, reading them back, attention of one query per sequence
// over it, and cutting sequences down to the tokens that attention used most.
#include <algorithm>
#include <cmath>

#include "serve_args.h"
#include "serve_device.h"

namespace simp {
namespace {

// A simp_rt_kv8 as the kernels take it: device addresses, the block as a shift.
struct Cache {
  int8_t *k, *v;
  float *ks, *vs;
  int64_t st_seq, st_head, st_token, sc_seq, sc_head;
  int n, hk, cap, hs, shift;
};

__device__ __forceinline__ int64_t clampl(int64_t x, int64_t lo, int64_t hi) {
  return x < lo ? lo : x > hi ? hi : x;
}

// max that a NaN comes through
__device__ __forceinline__ float max_nan(float a, float b) { return a != a || a > b ? a : b; }

__device__ __forceinline__ uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
  return __builtin_amdgcn_perm(hi, lo, sel);  // bytes 0-3 of lo, 4-7 of hi
}

// Nearest code to x / s, ties to even, of the exact quotient; s > 0 and finite, inv =
// 1 / s rounded (or anything near it).  x - n s is exact where n is next to the
// quotient: n has 7 bits, and what remains is a multiple of the last bit of s / 2 below s.
__device__ __forceinline__ int code_of(float x, float s, float inv) {
  const float n = rintf(fminf(fmaxf(x * inv, -127.f), 127.f));
  const float r = fmaf(-n, s, x), half = 0.5f * s, a = fabsf(r);
  const bool odd = ((int)n & 1) != 0;
  const float to = r < 0.f ? n - 1.f : n + 1.f;  // the other neighbour
  return (int)fminf(fmaxf(a > half || (a == half && odd) ? to : n, -127.f), 127.f);
}

// The codes of four numbers, in bytes.  The sum of x inv with 1.5 2^23 has the nearest
// whole number in its low bits, and x inv is within 127 2^-24 of the quotient: only
// where it comes that close to the middle of two codes does the exact way decide.
__device__ __forceinline__ uint32_t codes4(const float4 &x, float s, float inv) {
  constexpr float kShift = 12582912.f;
  const float a = fmaf(x.x, inv, kShift), b = fmaf(x.y, inv, kShift);
  const float c = fmaf(x.z, inv, kShift), d = fmaf(x.w, inv, kShift);
  const float off = fmaxf(fmaxf(fabsf(fmaf(x.x, inv, kShift - a)), fabsf(fmaf(x.y, inv, kShift - b))),
                          fmaxf(fabsf(fmaf(x.z, inv, kShift - c)), fabsf(fmaf(x.w, inv, kShift - d))));
  uint32_t r[4] = {__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d)};
  if (off > 0.4999f) {
    r[0] = (uint32_t)code_of(x.x, s, inv);
    r[1] = (uint32_t)code_of(x.y, s, inv);
    r[2] = (uint32_t)code_of(x.z, s, inv);
    r[3] = (uint32_t)code_of(x.w, s, inv);
  }
  return perm(perm(r[3], r[2], 0x0c0c0400), perm(r[1], r[0], 0x0c0c0400), 0x05040100);
}

// i / n by way of per = ceil(2^20 / n): exact for i < 4096 n (n up to 64).
inline uint32_t per_of(int64_t n) { return (uint32_t)cdiv(int64_t(1) << 20, n); }
__device__ __forceinline__ int over(int i, uint32_t per) { return (int)((uint32_t)i * per >> 20); }

// Four codes times ratio <= 1 (a NaN never: the caller clears those), rounded to the
// nearest, ties to even: the sum with 1.5 2^52 has the rounded number in its low bits.
__device__ __forceinline__ uint32_t rescale4(uint32_t c, double ratio) {
  uint32_t r[4];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const double t = fma((double)(int)(int8_t)(c >> (8 * e)), ratio, 6755399441055744.0);
    r[e] = (uint32_t)__double_as_longlong(t);
  }
  return perm(perm(r[3], r[2], 0x0c0c0400), perm(r[1], r[0], 0x0c0c0400), 0x05040100);
}

// ---------------------------------------------------------------- append
//
// One block of one head, K or V (blockIdx.z), to a block of threads that holds the
// new rows in registers between their maximum and their codes (kAppendChunks times four
// values to a thread): x is read once.  Sequence b has the slots starts[b] / T + 2 b and
// on: n rows touch at most n / T + 2 blocks.
// 7688 rows of 8 heads, 128 wide: 23.4 us for 79 MB, 3.4 TB/s of the 4.9 that a large copy
// reaches (28.7 us with the exact quotient of every value and a division for each row
// number; 50 us when x was read twice): the loads of a block end before its codes begin, and
// only other blocks fill the time.  One row of 32 sequences: 3.8 us, the latency of
// starts, rows and scale in turn.

struct AppendArgs {
  Cache c;
  const float *k, *v;
  const int *starts, *lengths;
  int64_t k_row, k_head, v_row, v_head;
  int rows;
  uint32_t per;  // of head_size / 4
};

constexpr int kAppendChunks = 8;

template <int THREADS, bool VEC>
__global__ void __launch_bounds__(THREADS) kv8_append_k(const AppendArgs a) {
  __shared__ float top_s[THREADS / 64];
  const Cache &c = a.c;
  const int t = blockIdx.x, h = blockIdx.y, T = 1 << c.shift, tid = threadIdx.x;
  const int b = last_of(c.n, [&](int s) { return (clampi(a.starts[s], 0, a.rows) >> c.shift) + 2 * s <= t; });
  const int r0 = clampi(a.starts[b], 0, a.rows), r1 = clampi(a.starts[b + 1], r0, a.rows);
  const int64_t end = a.lengths[b], have = end - (r1 - r0);  // positions of the new rows
  const int64_t from = clampl(have, 0, c.cap), to = clampl(end, 0, c.cap);
  const int slot0 = (r0 >> c.shift) + 2 * b;
  const int64_t blk = (from >> c.shift) + (t - slot0);
  const int64_t p0 = blk << c.shift;
  if (t < slot0 || from >= to || p0 >= to) return;
  const int64_t p1 = p0 + T < to ? p0 + T : to;
  const int64_t first = p0 > from ? p0 : from;  // tokens p0 .. first-1 are there already
  const bool is_v = blockIdx.z != 0;
  const int64_t row = is_v ? a.v_row : a.k_row;
  const float *x = (is_v ? a.v + h * a.v_head : a.k + h * a.k_head) + (r0 + first - have) * row;
  int8_t *codes = (is_v ? c.v : c.k) + b * c.st_seq + h * c.st_head + p0 * c.st_token;
  float *sc = (is_v ? c.vs : c.ks) + b * c.sc_seq + h * c.sc_head + blk;
  const int quads = c.hs >> 2, old = (int)(first - p0), nw = (int)(p1 - first) * quads;
  const float before = old ? *sc : 0.f;

  float4 v[kAppendChunks];
  float top = 0.f;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < kAppendChunks; i++) {
    const int e = tid + i * THREADS;
    v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (e < nw) {
      const int r = over(e, a.per);
      const float *p = x + r * row + 4 * (e - r * quads);
      if (VEC) v[i] = *(const float4 *)p;
      else v[i] = make_float4(p[0], p[1], p[2], p[3]);
    }
  }
#pragma unroll
  for (int i = 0; i < kAppendChunks; i++) {
    const float m = fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
    top = fmaxf(top, m);
    const float z = v[i].x * 0.f + v[i].y * 0.f + v[i].z * 0.f + v[i].w * 0.f;
    odd |= z != 0.f;  // of an infinity or NaN
  }
  top = wave_max_dpp(top);
  if (__any(odd)) top = NAN;
  if ((tid & 63) == 0) top_s[tid >> 6] = top;
  __syncthreads();  // also: every thread has read the scale
#pragma unroll
  for (int i = 0; i < THREADS / 64; i++) top = max_nan(top, top_s[i]);
  const float s = max_nan(before, top / 127.f);
  const bool live = s > 0.f && s < INFINITY;
  if (old && !(before == s)) {  // what the block held, to the new scale
    const double ratio = live ? (double)before / (double)s : 0.0;
    for (int e = tid; e < old * quads; e += THREADS) {
      const int r = over(e, a.per);
      uint32_t *p = (uint32_t *)(codes + r * c.st_token + 4 * (e - r * quads));
      *p = live ? rescale4(*p, ratio) : 0u;
    }
  }
  const float inv = live ? 1.f / s : 0.f;
  const bool tiny = live && s < 1e-37f;  // 1 / s may be infinite or coarse
#pragma unroll
  for (int i = 0; i < kAppendChunks; i++) {
    const int e = tid + i * THREADS;
    if (e < nw) {
      const int r = over(e, a.per);
      uint32_t q = 0;
      if (tiny) {
        const float y[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int w = 0; w < 4; w++)
          q |= (uint32_t)(uint8_t)(int8_t)(int)fmin(fmax(rint((double)y[w] / (double)s), -127.0), 127.0) << (8 * w);
      } else if (live) {
        q = codes4(v[i], s, inv);
      }
      *(uint32_t *)(codes + (old + r) * c.st_token + 4 * (e - r * quads)) = q;
    }
  }
  if (tid == 0) *sc = s;
}

// ------------------------------------------------------------------ read

struct ReadArgs {
  Cache c;
  const int *starts, *lengths;
  float *k, *v;
  int64_t k_row, k_head, v_row, v_head;
  int rows;
};

constexpr int kReadRows = 32;

// kReadRows packed rows of one head, K and V.  7688 rows of 8 heads, 128 wide: 15-18 us
// for 79 MB, 4.4-5.2 TB/s; memory bounds it.
template <bool VEC>
__global__ void __launch_bounds__(256) kv8_read_k(const ReadArgs a) {
  __shared__ int64_t at[kReadRows];  // the token's codes; -1: zeros; -2: nobody's row
  __shared__ float ks[kReadRows], vs[kReadRows];
  const Cache &c = a.c;
  const int first = blockIdx.x * kReadRows, h = blockIdx.y, n = min(kReadRows, a.rows - first);
  if (threadIdx.x < 64) {
    const int r = first + min((int)threadIdx.x, n - 1);
    int b = last_of(c.n, [&](int s) { return clampi(a.starts[s], 0, a.rows) <= first; });
    for (int hi = c.n - 1; b < hi && clampi(a.starts[b + 1], 0, a.rows) <= r;) {  // this row's
      const int mid = (b + hi + 1) >> 1;
      if (clampi(a.starts[mid], 0, a.rows) <= r) b = mid;
      else hi = mid - 1;
    }
    const int r0 = clampi(a.starts[b], 0, a.rows), r1 = clampi(a.starts[b + 1], r0, a.rows);
    if ((int)threadIdx.x < n) {
      const int64_t p = (int64_t)a.lengths[b] - (r1 - r);
      const bool mine = r >= r0 && r < r1, in = p >= 0 && p < c.cap;
      at[threadIdx.x] = !mine ? -2 : !in ? -1 : b * c.st_seq + h * c.st_head + p * c.st_token;
      const int64_t z = b * c.sc_seq + h * c.sc_head + (p >> c.shift);
      ks[threadIdx.x] = mine && in ? c.ks[z] : 0.f;
      vs[threadIdx.x] = mine && in ? c.vs[z] : 0.f;
    }
  }
  __syncthreads();
  const int quads = c.hs >> 2;
#pragma unroll 4
  for (int e = threadIdx.x; e < n * quads; e += 256) {
    const int i = e / quads, d = 4 * (e - i * quads);
    const int64_t o = at[i];
    if (o == -2) continue;
    const uint32_t kc = o < 0 ? 0u : *(const uint32_t *)(c.k + o + d);
    const uint32_t vc = o < 0 ? 0u : *(const uint32_t *)(c.v + o + d);
    float *kd = a.k + (int64_t)(first + i) * a.k_row + h * a.k_head + d;
    float *vd = a.v + (int64_t)(first + i) * a.v_row + h * a.v_head + d;
    float x[4], y[4];
#pragma unroll
    for (int w = 0; w < 4; w++) {
      x[w] = (float)(int8_t)(kc >> (8 * w)) * ks[i];
      y[w] = (float)(int8_t)(vc >> (8 * w)) * vs[i];
    }
    if (VEC) {
      *(float4 *)kd = make_float4(x[0], x[1], x[2], x[3]);
      *(float4 *)vd = make_float4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
      for (int w = 0; w < 4; w++) {
        kd[w] = x[w];
        vd[w] = y[w];
      }
    }
  }
}

// ------------------------------------------------------------- attention
//
// Both products run on v_mfma_i32_16x16x64_i8 with the codes as they lie in memory:
// the other factor (q, then the weights) is rounded to a whole number of 24 bits of
// its largest element and taken apart into three signed bytes, v = l0 + 256 l1 +
// 65536 l2, so every product and sum is exact and the fp32 work is one combination
// of three integers.  Memory bounds the kernel (2 head_size bytes a token and kv head);
// converting the codes to floating point would cost more VALU time than that.
//   * A wave takes 64 tokens at a time.  S^T = K Q^T: lane (i, g) = (lane % 16, lane /
//     16) loads 16 codes of token i, and ends with the scores of tokens 16 t + 4 g + r
//     (t, r < 4) for query head i of the group.
//   * O^T = V^T P^T: the order of the 64 tokens inside the product is free as long as
//     both factors have it, so lane group g takes the tokens 16 t + 4 g + r, whose
//     weights it holds already, and the V rows it loads 4 codes at a time are turned
//     by 4x4 byte transposes in registers.  Neither product touches LDS.
//   * The head dimension is free in the same way: row i of the n-th product of a
//     64-dimension chunk is d = 4 i + n.
// Weights: p = 2^(s - m) of the tile's own maximum m, times the V block's scale over the
// tile's largest; the integer's unit is the largest of these products / 8.35e6, so
// that each tile keeps 24 bits of what it contributes, whatever the scales.
// A block of four waves takes a piece of one kv head's tokens, its tiles in turn; the
// rest of a row's softmax is joined by kv8_join_k.
// 131072 tokens of 8 heads, 128 wide: 57 us for 268 MB of codes, 4.7 TB/s, and 17 MB of scores.
// 16 sequences of 1 to 4096 tokens: 16 us for 57 MB, 3.6 TB/s (19.6 with pieces of one length
// for each sequence's place in the grid, whose empty blocks leave CUs with two full
// ones next to idle ones; 26 with exactly equal shares, which span sequences); half of it is the
// latency of lengths, q and the first tile, and of the join of the waves.

typedef int v4i __attribute__((ext_vector_type(4)));

struct AttnArgs {
  Cache c;
  const float *q;
  const int *lengths;
  float *out;
  const float *seen_in;
  float *seen_out;
  int64_t q_seq, q_head, o_seq, o_head, si_seq, si_head, so_seq, so_head;
  int heads, group;
  int sets, width;    // sets of up to `width` (at most 16) query heads of a kv head
  int blocks;         // that full pieces should come to
  float scale;        // times log2(e): the scores are powers of two
  float *scores;      // [n, heads, score_row], or null
  int64_t score_row;  // the capacity in whole tiles of 64
  float *part;        // [units' first pieces, width, pieces of a unit, head_size], unnormalised
  float2 *stat;       // the same without head_size: maximum and sum
  int *starts;        // [n + 2]: pieces of a unit in the sequences before; the share (n > 64)
};

// Sums of whole numbers over the wave, and running sums over its lanes.
__device__ __forceinline__ int wave_scan(int x) {
  const int lane = threadIdx.x & 63;
  // within rows of 16 lanes (lanes without a neighbour add 0), then the rows before
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  const int a = __builtin_amdgcn_readlane(x, 15), b = __builtin_amdgcn_readlane(x, 31), c = __builtin_amdgcn_readlane(x, 47);
  return x + (lane < 16 ? 0 : lane < 32 ? a : lane < 48 ? a + b : a + b + c);
}
__device__ __forceinline__ int wave_total(int scanned) { return __builtin_amdgcn_readlane(scanned, 63); }

// The work: rounds of 256 tokens (a tile for each wave).  A piece is up to `share` rounds of
// one unit (a set of the query heads of a kv head, of one sequence), with a share that makes
// about `blocks` pieces of all, whatever the lengths.  Pieces follow each other sequence
// after sequence, and in a sequence unit after unit; block i has piece i.  Up to 64
// sequences, one to a lane, are counted by every wave for itself; more by kv8_plan_k.
constexpr int kRound = 256;
__device__ __forceinline__ int rounds_of(const AttnArgs &a, int b) {
  return b < a.c.n ? (clampi(a.lengths[b], 0, a.c.cap) + kRound - 1) / kRound : 0;
}
__device__ __forceinline__ int share_of(const AttnArgs &a, int rounds) {
  return max((rounds * (a.c.hk * a.sets) + a.blocks - 1) / a.blocks, 1);
}
struct Piece {
  int b, unit;       // sequence, unit in it
  int place, count;  // among the unit's pieces
  int share;
};
__device__ __forceinline__ bool find_piece(const AttnArgs &a, int x, Piece &p) {
  const int lane = threadIdx.x & 63, n = a.c.n, units = a.c.hk * a.sets;
  int before;
  if (n <= 64) {
    const int r = rounds_of(a, lane);
    p.share = share_of(a, wave_total(wave_scan(r)));
    const int own = (r + p.share - 1) / p.share, upto = wave_scan(own);
    if (x == 0 && threadIdx.x < 64) {  // for kv8_join_k
      if (lane < n) a.starts[lane + 1] = upto;
      if (lane == 0) a.starts[0] = 0;
    }
    const unsigned long long who = __ballot(upto > x / units);
    if (!who) return false;
    p.b = __ffsll(who) - 1;
    p.count = __builtin_amdgcn_readlane(own, p.b);
    before = __builtin_amdgcn_readlane(upto, p.b) - p.count;
  } else {
    const auto *starts = (const __attribute__((address_space(4))) int *)a.starts;
    p.share = starts[n + 1];
    if (starts[n] <= x / units) return false;
    p.b = last_of(n, [&](int s) { return a.starts[s] <= x / units; });
    before = starts[p.b];
    p.count = starts[p.b + 1] - before;
  }
  const int y = x - before * units;
  p.unit = y / p.count;
  p.place = y - p.unit * p.count;
  return true;
}

// The pieces of a unit in the sequences before each of more than 64, and in all; then the
// share.  65 sequences: 2.4 us and 14.9 for kv8_attn_k, against 15.9 where its waves count for
// themselves; 200: 3-5 and 36.9 against 38.5; 1024: 3-5 and 24 against 59.
__global__ void __launch_bounds__(1024) kv8_plan_k(const AttnArgs a) {
  __shared__ int wave_s[2][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = a.c.n;
  // the running sum of x over the block's threads, and its total
  const auto block_scan = [&](int x, int slot, int &total) {
    x = wave_scan(x);
    if (lane == 63) wave_s[slot][wave] = x;
    __syncthreads();
    const int waves = wave_scan(lane < 16 ? wave_s[slot][lane] : 0);
    total = __builtin_amdgcn_readlane(waves, 15);
    return x + (wave ? __builtin_amdgcn_readlane(waves, wave - 1) : 0);
  };
  int rounds = 0, total;
  for (int b = tid; b < n; b += 1024) rounds += rounds_of(a, b);
  block_scan(rounds, 0, total);
  const int share = share_of(a, total);
  int before = 0, slot = 1;
  for (int b0 = 0; b0 < n; b0 += 1024, slot ^= 1) {
    const int upto = before + block_scan((rounds_of(a, b0 + tid) + share - 1) / share, slot, total);
    if (b0 + tid < n) a.starts[b0 + tid + 1] = upto;
    before += total;
  }
  if (tid == 0) {
    a.starts[0] = 0;
    a.starts[n + 1] = share;
  }
}

constexpr float kUnit = 8.35e6f;        // v + 0x808080 stays below 2^24 and above 0
constexpr uint32_t kBytes = 0x808080u;  // makes the three bytes unsigned

// The three byte planes of four numbers v + kBytes (bits above 24 are ignored).
__device__ __forceinline__ void planes(const uint32_t (&u)[4], uint32_t &l0, uint32_t &l1, uint32_t &l2) {
  const uint32_t a = perm(u[1], u[0], 0x05010400), b = perm(u[3], u[2], 0x05010400);
  l0 = perm(b, a, 0x05040100) ^ 0x80808080u;
  l1 = perm(b, a, 0x07060302) ^ 0x80808080u;
  l2 = perm(perm(u[3], u[2], 0x0c0c0602), perm(u[1], u[0], 0x0c0c0602), 0x05040100) ^ 0x80808080u;
}

// 4x4 bytes: out[n] = byte n of in[0..3]
__device__ __forceinline__ void turn4(const uint32_t (&in)[4], uint32_t (&out)[4]) {
  const uint32_t a = perm(in[1], in[0], 0x05010400), b = perm(in[1], in[0], 0x07030602);
  const uint32_t c = perm(in[3], in[2], 0x05010400), d = perm(in[3], in[2], 0x07030602);
  out[0] = perm(c, a, 0x05040100);
  out[1] = perm(c, a, 0x07060302);
  out[2] = perm(d, b, 0x05040100);
  out[3] = perm(d, b, 0x07060302);
}

// max / sum over the four lanes with the same lane % 16
__device__ __forceinline__ float quad_max(float v) {
  float a = v, b = v;
  permlane16_swap(a, b);
  a = b = fmaxf(a, b);
  permlane32_swap(a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float quad_sum(float v) {
  float a = v, b = v;
  permlane16_swap(a, b);
  a = b = a + b;
  permlane32_swap(a, b);
  return a + b;
}

// 16 bytes from a 4-byte boundary
__device__ __forceinline__ void load16(void *to, const void *p) {
  __builtin_memcpy(to, __builtin_assume_aligned(p, 4), 16);
}

// The sum over the four lanes of a quad.
__device__ __forceinline__ float quad_add(float v) {
  v += dpp_mov<kDppXor1>(v);
  return v + dpp_mov<kDppXor2>(v);
}

// NC: 64-dimension chunks of a head.  QUAD: up to four query heads, lane i of the 16
// columns with byte i % 4 of head i / 4 (the fourth of them nothing), so that one
// product does what three do with the bytes apart, one byte plane is kept instead of
// three, and a sum over the quad joins them; else up to 16 heads, a column each.
template <int NC, bool QUAD>
__global__ void __launch_bounds__(256, NC == 1 ? 4 : NC == 2 && QUAD ? 3 : NC < 4 ? 2 : 1)
    kv8_attn_k(const AttnArgs a) {
  extern __shared__ float lds[];  // o [4][cols][hs], then m and l [4][cols]
  constexpr int L = QUAD ? 1 : 3;
  const Cache &c = a.c;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i16 = lane & 15, g = lane >> 4, hs = c.hs;
  const int head = QUAD ? i16 >> 2 : i16, byte = QUAD ? i16 & 3 : 0;  // of the lane's column
  Piece piece;
  if (!find_piece(a, (int)blockIdx.x, piece)) return;
  const int b = piece.b, hk = piece.unit / a.sets, set0 = (piece.unit - hk * a.sets) * a.width;
  const int cols = min(a.width, a.group - set0), h0 = hk * a.group + set0;  // query heads h0 ..
  const int len = clampi(a.lengths[b], 0, c.cap), chunk = piece.share * kRound;
  const int from = piece.place * chunk, to = len - from < chunk ? len : from + chunk;
  const int8_t *kp = c.k + b * c.st_seq + hk * c.st_head;
  const int8_t *vp = c.v + b * c.st_seq + hk * c.st_head;
  const float *ksp = c.ks + b * c.sc_seq + hk * c.sc_head, *vsp = c.vs + b * c.sc_seq + hk * c.sc_head;
  // What takes the lane's byte of two numbers, makes it signed, and its weight.
  const uint32_t pick = byte == 3 ? 0x0c0c0c0cu : 0x0c0c0400u + 0x0101u * byte;
  const uint32_t flip = byte == 3 ? 0u : 0x80808080u;
  const float weight = byte == 0 ? 1.f : byte == 1 ? 256.f : byte == 2 ? 65536.f : 0.f;
  auto bytes_of = [&](const uint32_t (&u)[4], uint32_t (&l)[L]) {
    if constexpr (QUAD) l[0] = perm(perm(u[3], u[2], pick), perm(u[1], u[0], pick), 0x05040100) ^ flip;
    else planes(u, l[0], l[1], l[2]);
  };
  // The number that a column's products stand for (the lane's byte's part of it).
  auto number = [&](const v4i (&x)[L], int r) {
    if constexpr (QUAD) return (float)x[0][r] * weight;
    else return fmaf((float)x[2][r], 65536.f, (float)(x[1][r] * 256 + x[0][r]));
  };

  // The head's dimensions as the lane's K loads have them: 16 from doff on, of which
  // those below 64 j + 16 g belong to the chunk before (the row's end).
  uint32_t doff[NC];
  v4i ql[NC][L];
  float qf;  // times 2^qe: what a unit of q's whole numbers is worth
  int qe;
  {
    float x[NC][16], top = 0.f;
    bool odd = false;
    const float *qr = a.q + b * a.q_seq + (h0 + min(head, cols - 1)) * a.q_head;
#pragma unroll
    for (int j = 0; j < NC; j++) {
      doff[j] = (uint32_t)min(64 * j + 16 * g, hs - 16);
#pragma unroll
      for (int e = 0; e < 16; e += 4) load16(&x[j][e], qr + doff[j] + e);
    }
#pragma unroll
    for (int j = 0; j < NC; j++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        odd |= !(fabsf(x[j][e]) < INFINITY);
        if ((int)doff[j] + e < 64 * j + 16 * g) x[j][e] = 0.f;
        top = fmaxf(top, fabsf(x[j][e]));
      }
    top = quad_max(top);
    const unsigned long long who = __ballot(odd);  // a query that is not finite: its row is NaN
    if ((who >> i16) & 0x0001000100010001ull) top = NAN;
    // by way of [1, 2): 1 / top alone may be too large, and top / kUnit subnormal
    const int e2 = top > 0.f ? -ilogbf(top) : 0;
    const float top1 = ldexpf(top, e2);
    const float inv = top > 0.f ? kUnit / top1 : 0.f;
    qf = top1 * a.scale * (8388608.f / kUnit);  // over 2^qe
    qe = -23 - e2;
#pragma unroll
    for (int j = 0; j < NC; j++)
#pragma unroll
      for (int w = 0; w < 4; w++) {
        uint32_t u[4], l[L];
#pragma unroll
        for (int r = 0; r < 4; r++)
          u[r] = (uint32_t)(__float2int_rn(ldexpf(x[j][4 * w + r], e2) * inv) + (int)kBytes);
        bytes_of(u, l);
#pragma unroll
        for (int i = 0; i < L; i++) ql[j][i][w] = (int)l[i];
      }
  }
  const int last = to - 1;  // rows behind it repeat it, and are masked
  // Addresses: a wave-uniform base for the tile, and 24-bit row numbers times strides
  // below 2^24 (the caller sees to that).
  const uint32_t stride = (uint32_t)c.st_token;
  v4i kf[4][NC];
  uint32_t vf[4][NC][4];
  auto load_k = [&](int key0) {
    const int8_t *base = kp + (int64_t)key0 * c.st_token;
    const uint32_t lim = (uint32_t)(last - key0);
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const uint32_t row = __umul24(min((uint32_t)(16 * t + i16), lim), stride);
#pragma unroll
      for (int j = 0; j < NC; j++) load16(&kf[t][j], base + (row + doff[j]));
    }
  };
  auto load_v = [&](int key0) {
    const int8_t *base = vp + (int64_t)key0 * c.st_token;
    const uint32_t lim = (uint32_t)(last - key0);
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const uint32_t row = __umul24(min((uint32_t)(16 * t + 4 * g + r), lim), stride);
#pragma unroll
        for (int j = 0; j < NC; j++)
          vf[t][j][r] = *(const uint32_t *)(base + (row + (uint32_t)min(64 * j + 4 * i16, hs - 4)));
      }
  };

  if (from + 64 * wave < to) load_k(from + 64 * wave);
  float o[NC][4][4];  // [j][n][r]: d = 64 j + 16 g + 4 r + n
#pragma unroll
  for (int j = 0; j < NC; j++)
#pragma unroll
    for (int n = 0; n < 4; n++)
#pragma unroll
      for (int r = 0; r < 4; r++) o[j][n][r] = 0.f;
  float m = -INFINITY, l = 0.f;
  float *scores = a.scores ? a.scores + ((int64_t)b * a.heads + h0 + min(head, cols - 1)) * a.score_row + 4 * g
                           : nullptr;
  const bool keeper = head < cols && byte == 0;  // writes what its column's lanes agree on
  for (int key0 = from + 64 * wave; key0 < to; key0 += 256) {
    load_v(key0);
    float ks[4], vs[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const int blk = min(key0 + 16 * t, last) >> c.shift;
      ks[t] = ksp[blk];
      vs[t] = vsp[blk];
    }
    // scores
    const int left = to - key0 - 4 * g;  // tokens 16 t + r below it are there
    float s[4][4];
    float mt = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; t++) {
      v4i x[L];
#pragma unroll
      for (int i = 0; i < L; i++) x[i] = v4i{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < NC; j++)
#pragma unroll
        for (int i = 0; i < L; i++)
          x[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[t][j], ql[j][i], x[i], 0, 0, 0);
      const float f = ldexpf(qf * ks[t], qe);
#pragma unroll
      for (int r = 0; r < 4; r++) {
        float y = number(x, r);
        if (QUAD) y = quad_add(y);
        s[t][r] = 16 * t + r < left ? y * f : -INFINITY;
        mt = fmaxf(mt, s[t][r]);
      }
    }
    load_k(min(key0 + 256, last));  // the next tile's, on their way during this one's V
    if (scores && keeper) {  // score rows are padded to whole tiles
#pragma unroll
      for (int t = 0; t < 4; t++)
        *(float4 *)(scores + key0 + 16 * t) = make_float4(s[t][0], s[t][1], s[t][2], s[t][3]);
    }
    mt = quad_max(mt);
    const float mu = mt == -INFINITY ? 0.f : mt;
    // weights
    const float vsum = (vs[0] + vs[1]) + (vs[2] + vs[3]);
    const float vtop = fmaxf(fmaxf(vs[0], vs[1]), fmaxf(vs[2], vs[3]));
    const int ve = vtop > 0.f ? ilogbf(vtop) : 0;  // the scales over 2^ve lie below 2
    float w[4][4], lt = 0.f, wt = 0.f;
#pragma unroll
    for (int t = 0; t < 4; t++) {
      const float vr = ldexpf(vs[t], -ve);
#pragma unroll
      for (int r = 0; r < 4; r++) {
        const float p = 16 * t + r < left ? pow2(s[t][r] - mu) : 0.f;
        lt += p;
        w[t][r] = p * vr;
        wt = fmaxf(wt, w[t][r]);
      }
    }
    wt = fmaxf(quad_max(wt), 1e-30f);
    const float inv = kUnit * __builtin_amdgcn_rcpf(wt);
    v4i wl[L];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      uint32_t u[4], y[L];
#pragma unroll
      for (int r = 0; r < 4; r++)  // the sum with 2^23 has the rounded number in its low bits
        u[r] = __float_as_uint(fmaf(w[t][r], inv, 8388608.f)) + kBytes;
      bytes_of(u, y);
#pragma unroll
      for (int i = 0; i < L; i++) wl[i][t] = (int)y[i];
    }
    const float mn = fmaxf(m, mt), mnu = mn == -INFINITY ? 0.f : mn;
    const float alpha = pow2(m - mnu), beta = pow2(mt - mnu);
    m = mn;
    l = fmaf(l, alpha, lt * beta);
    float f = ldexpf(beta * wt * (1.f / kUnit), ve);
    if (!(vsum < INFINITY)) f = NAN;  // a block that is not finite: the row is NaN
    if (QUAD) f *= weight;
#pragma unroll
    for (int j = 0; j < NC; j++) {
      v4i vt[4];
#pragma unroll
      for (int t = 0; t < 4; t++) {
        uint32_t x[4];
        turn4(vf[t][j], x);
#pragma unroll
        for (int n = 0; n < 4; n++) vt[n][t] = (int)x[n];
      }
#pragma unroll
      for (int n = 0; n < 4; n++) {
        v4i x[L];
#pragma unroll
        for (int i = 0; i < L; i++)
          x[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vt[n], wl[i], v4i{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const float y = QUAD ? (float)x[0][r] : number(x, r);
          o[j][n][r] = fmaf(y, f, o[j][n][r] * alpha);
        }
      }
    }
  }
  // the four waves' rows together
  l = quad_sum(l);
  float *ml = lds + 4 * cols * hs;
  float *row = lds + (wave * cols + min(head, cols - 1)) * hs;
#pragma unroll
  for (int j = 0; j < NC; j++)
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int d = 64 * j + 16 * g + 4 * r;
      float4 x = make_float4(o[j][0][r], o[j][1][r], o[j][2][r], o[j][3][r]);
      if (QUAD) x = make_float4(quad_add(x.x), quad_add(x.y), quad_add(x.z), quad_add(x.w));
      if (keeper && d < hs) *(float4 *)(row + d) = x;
    }
  if (keeper && g == 0) {
    ml[wave * cols + head] = m;
    ml[(4 + wave) * cols + head] = l;
  }
  __syncthreads();
  const int quads = hs >> 2;
  for (int e = threadIdx.x; e < cols * quads; e += 256) {
    const int col = e / quads, d = 4 * (e - col * quads);
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) M = fmaxf(M, ml[w * cols + col]);
    const float mu = M == -INFINITY ? 0.f : M;
    float sum = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float f = pow2(ml[w * cols + col] - mu);
      const float4 y = *(const float4 *)(lds + (w * cols + col) * hs + d);
      sum = fmaf(f, ml[(4 + w) * cols + col], sum);
      x.x = fmaf(f, y.x, x.x);
      x.y = fmaf(f, y.y, x.y);
      x.z = fmaf(f, y.z, x.z);
      x.w = fmaf(f, y.w, x.w);
    }
    const int64_t at = ((int64_t)blockIdx.x - piece.place) * a.width + (int64_t)col * piece.count + piece.place;
    *(float4 *)(a.part + at * hs + d) = x;
    if (d == 0) a.stat[at] = make_float2(M, sum);
  }
}

// 16 sequences of up to 4096 tokens, 32 heads, with the accumulated weights: 4.8 us;
// 131072 tokens of one: 8 us for 25 MB.
// The chunks of a row together.  blockIdx.x below the group: that query head's row of
// out, head_size / 4 threads to a chunk and as many chunks at a time as there are
// threads; above: TILE tokens of the accumulated weights.
template <int TILE>
__global__ void __launch_bounds__(256) kv8_join_k(const AttnArgs a) {
  extern __shared__ float lds[];
  __shared__ float4 so[256];
  __shared__ float top_s[4], sum_s[4];
  const Cache &c = a.c;
  const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int len = clampi(a.lengths[b], 0, c.cap);
  const auto *starts = (const __attribute__((address_space(4))) int *)a.starts;  // a scalar load
  const int before = starts[b], ns = starts[b + 1] - before, hs = c.hs, wd = a.width;
  const int64_t first = ((int64_t)before * c.hk * a.sets) + (int64_t)hk * a.sets * ns;
  // A head's first row.
  const auto row_of = [&](int g) {
    const int set = g / wd;
    return (first + (int64_t)set * ns) * wd + (int64_t)(g - set * wd) * ns;
  };
  if ((int)blockIdx.x < a.group) {
    const int h = hk * a.group + blockIdx.x;
    float *out = a.out + b * a.o_seq + h * a.o_head;
    if (len == 0) {
      for (int d = tid; d < hs; d += 256) out[d] = 0.f;
      return;
    }
    const float2 *st = a.stat + row_of(blockIdx.x);
    const float *part = a.part + row_of(blockIdx.x) * hs;
    float M = -INFINITY;
    for (int s = tid; s < ns; s += 256) M = fmaxf(M, st[s].x);
    M = wave_max_dpp(M);
    if (lane == 0) top_s[wave] = M;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; w++) M = fmaxf(M, top_s[w]);
    const float mu = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    for (int s = tid; s < ns; s += 256) {
      const float2 ml = st[s];
      const float f = pow2(ml.x - mu);
      lds[s] = f;
      L = fmaf(f, ml.y, L);
    }
    L = wave_sum_dpp(L);
    if (lane == 0) sum_s[wave] = L;
    __syncthreads();
    const int quads = hs >> 2, rows = 256 / quads, r = tid / quads, q = tid - r * quads;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < rows) {
#pragma unroll 4
      for (int s = r; s < ns; s += rows) {
        const float f = lds[s];
        const float4 y = *(const float4 *)(part + (int64_t)s * hs + 4 * q);
        x.x = fmaf(f, y.x, x.x);
        x.y = fmaf(f, y.y, x.y);
        x.z = fmaf(f, y.z, x.z);
        x.w = fmaf(f, y.w, x.w);
      }
    }
    so[tid] = x;
    __syncthreads();
    for (int d = tid; d < hs; d += 256) {
      float s = 0.f, l = 0.f;
      for (int i = 0; i < min(rows, ns); i++) s += ((const float *)so)[4 * (i * quads + (d >> 2)) + (d & 3)];
#pragma unroll
      for (int w = 0; w < 4; w++) l += sum_s[w];
      out[d] = s / l;
    }
    return;
  }
  const int t0 = ((int)blockIdx.x - a.group) * TILE;
  if (t0 >= len) return;
  // A thread has the tokens t0 + tid and 256 on.  What it adds to and up to four heads'
  // scores are asked for first: the pieces' sums take their time meanwhile.
  constexpr int kMine = TILE / 256, kAhead = 4;
  const float *sc = a.scores + ((int64_t)b * a.heads + hk * a.group) * a.score_row;
  float was[kMine], ahead[kAhead][kMine];
#pragma unroll
  for (int i = 0; i < kMine; i++) {
    const int t = min(t0 + tid + 256 * i, len - 1);
    was[i] = a.seen_in[b * a.si_seq + hk * a.si_head + t];
#pragma unroll
    for (int g = 0; g < kAhead; g++) ahead[g][i] = sc[min(g, a.group - 1) * a.score_row + t];
  }
  for (int g = wave; g < a.group; g += 4) {  // each head's maximum and 1 / sum
    const float2 *st = a.stat + row_of(g);
    float M = -INFINITY, L = 0.f;
    for (int s = lane; s < ns; s += 64) M = fmaxf(M, st[s].x);
    M = wave_max_dpp(M);
    const float mu = M == -INFINITY ? 0.f : M;
    for (int s = lane; s < ns; s += 64) L = fmaf(pow2(st[s].x - mu), st[s].y, L);
    L = wave_sum_dpp(L);
    if (lane == 0) {
      lds[2 * g] = mu;
      lds[2 * g + 1] = 1.f / L;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kMine; i++) {
    const int t = t0 + tid + 256 * i;
    if (t >= len) break;
    float w = 0.f;
#pragma unroll
    for (int g = 0; g < kAhead; g++)
      if (g < a.group) w = fmaf(pow2(ahead[g][i] - lds[2 * g]), lds[2 * g + 1], w);
#pragma unroll 4
    for (int g = kAhead; g < a.group; g++)
      w = fmaf(pow2(sc[g * a.score_row + t] - lds[2 * g]), lds[2 * g + 1], w);
    a.seen_out[b * a.so_seq + hk * a.so_head + t] = was[i] + w;
  }
}

// ----------------------------------------------------------------- evict

struct EvictArgs {
  Cache c, to;
  const int *lengths;
  const float *seen;
  float *new_seen;
  int *kept;
  int64_t se_seq, se_head, ns_seq, ns_head, kp_seq, kp_head;
  int budget, recent;
  uint32_t per;  // of the words of a row that kv8_move_k takes at a time
};

// Unsigned order of the weights: NaN above all, both zeros alike.  None has the order 0.
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The tokens of a wave's run, [t0, t1): f(token, its weight, the weight's order, or 0 from
// `old` on).  Up to 512 of them (8192 of the sequence) are in registers; more are read
// again.  Sixteen waves share four SIMDs here, so every instruction of f counts.
struct Run {
  const float *seen;
  int t0, t1, old;
  bool held;
  float x[8];
  uint32_t u[8];
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    const int lane = threadIdx.x & 63;
    if (held) {
#pragma unroll
      for (int i = 0; i < 8; i++)
        if (t0 + 64 * i < t1) f(t0 + 64 * i + lane, x[i], u[i]);
    } else {
      for (int t = t0 + lane; t - lane < t1; t += 64) {
        const float y = t < t1 ? seen[t] : 0.f;
        f(t, y, t < min(old, t1) ? order_of(y) : 0u);
      }
    }
  }
};

// The place-from-the-top search of kv8_select_k: among the weights whose order agrees with `prefix` above bit `shift + BITS`, a histogram of the next BITS bits
// (hist is 0 before and after); then the bin that holds the need-th from the top.
// Returns it, and what is left to take from it in `need`, its size in `size`.
template <int BITS>
__device__ __forceinline__ uint32_t select_digit(const Run &run, uint32_t prefix, int shift,
                                                 int &need, int &size, int *hist, int *wave_s) {
  constexpr int BINS = 1 << BITS, PER = BINS / 1024;  // bins of a thread
  static_assert(PER * 1024 == BINS, "");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int above_bits = min(shift + BITS, 31);
  const uint32_t same = shift + BITS == 32 ? 0u : 0xFFFFFFFFu << above_bits;
  run.each([&](int, float, uint32_t u) {
    if (u && ((u ^ prefix) & same) == 0) atomicAdd(&hist[u >> shift & (BINS - 1)], 1);
  });
  __syncthreads();
  // thread t has the bins from the top: BINS - 1 - PER t and the PER - 1 below
  int h[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    int &bin = hist[BINS - 1 - PER * tid - i];
    h[i] = bin;
    bin = 0;
    sum += h[i];
  }
  int upto = wave_scan(sum);  // bins of this wave's threads up to this one's
  if (lane == 63) wave_s[wave] = upto;
  __syncthreads();
  const int waves = wave_scan(lane < 16 ? wave_s[lane] : 0);
  if (wave > 0) upto += __builtin_amdgcn_readlane(waves, wave - 1);
  int above = upto - sum;
  if (above < need && need <= upto) {  // one thread
    int i = 0;
    while (above + h[i] < need) above += h[i++];
    wave_s[16] = BINS - 1 - PER * tid - i;
    wave_s[17] = need - above;
    wave_s[18] = h[i];
  }
  __syncthreads();
  const uint32_t digit = (uint32_t)wave_s[16];
  need = wave_s[17];
  size = wave_s[18];
  return digit << shift;
}

// Which tokens of one head stay, by one block: the order of the last weight that
// does, 12 bits and twice 10 from the top, then the places.  Twelve bits first, so
// that the weights, which share few exponents, do not all add to the same few
// counters.  Each wave has a run of tokens: it counts those that stay (and those equal
// to the last one, of which the first ones do), and writes them behind the other waves'.
// 128 heads of up to 8192 tokens: 11 us on half of the CUs (17 with the orders formed anew
// in each pass and the weights read again for the writing): three searches with their
// atomics in LDS, the count and the writing follow each other, and the 16 waves' issue
// bounds each.
__global__ void __launch_bounds__(1024) kv8_select_k(const EvictArgs a) {
  __shared__ int hist[4096];
  __shared__ int wave_s[32], more_s[16], equal_s[16];
  const int hk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int len = clampi(a.lengths[b], 0, a.c.cap);
  const float *seen = a.seen + b * a.se_seq + hk * a.se_head;
  float *ns = a.new_seen + b * a.ns_seq + hk * a.ns_head;
  int *kept = a.kept + b * a.kp_seq + hk * a.kp_head;
  if (len <= a.budget) {
    for (int t = tid; t < a.budget; t += 1024) {
      kept[t] = t < len ? t : -1;
      if (t < len) ns[t] = seen[t];
    }
    return;
  }
  Run run;
  const int each = (len + 1023) / 1024 * 64;  // tokens of a wave
  run.seen = seen;
  run.t0 = min(wave * each, len);
  run.t1 = min(run.t0 + each, len);
  run.held = each <= 512;
  const int old = run.old = len - a.recent;  // candidates 0 .. old-1
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const int t = run.t0 + 64 * i + lane;
    run.x[i] = run.held && t < run.t1 ? seen[t] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < 8; i++) run.u[i] = run.t0 + 64 * i + lane < min(old, run.t1) ? order_of(run.x[i]) : 0u;
#pragma unroll
  for (int i = 0; i < 4; i++) hist[tid + 1024 * i] = 0;
  __syncthreads();
  int need = a.budget - a.recent;  // of which so many stay (fewer than there are)
  uint32_t last = 0xFFFFFFFFu;     // the order of the last one that stays,
  uint32_t mask = 0xFFFFFFFFu;     // in these bits
  if (need > 0) {
    int size;
    last = select_digit<12>(run, 0, 20, need, size, hist, wave_s);
    mask = 0xFFF00000u;
    if (size != need) {
      last |= select_digit<10>(run, last, 10, need, size, hist, wave_s);
      mask = 0xFFFFFC00u;
    }
    if (size != need) {
      last |= select_digit<10>(run, last, 0, need, size, hist, wave_s);
      mask = 0xFFFFFFFFu;
    }
  }
  // Above `high` an order is larger than the last one in its bits, and from `last` to it equal.
  const uint32_t high = last | ~mask, range = ~mask;
  int more = max(run.t1 - max(run.t0, old), 0), equal = 0;  // of the wave
  run.each([&](int, float, uint32_t u) {
    more += __popcll(__ballot(u > high));
    equal += __popcll(__ballot(u - last <= range));
  });
  if (lane == 0) {
    more_s[wave] = more;
    equal_s[wave] = equal;
  }
  __syncthreads();
  int eq = 0, place = 0;  // equal ones before this wave's; where it writes
  {
    const int m = lane < 16 ? more_s[lane] : 0, e = lane < 16 ? equal_s[lane] : 0;  // of a wave
    const int es = wave_scan(e), ps = wave_scan(m + min(e, max(need - (es - e), 0)));
    if (wave > 0) {
      eq = __builtin_amdgcn_readlane(es, wave - 1);
      place = __builtin_amdgcn_readlane(ps, wave - 1);
    }
  }
  const auto below = [](unsigned long long who) {  // lanes before this one
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
  };
  run.each([&](int t, float x, uint32_t u) {
    const bool same = u - last <= range;
    const unsigned long long be = __ballot(same);
    const bool keep = u > high || (t >= old && t < run.t1) || (same && eq + below(be) < need);
    const unsigned long long bk = __ballot(keep);
    const int k = place + below(bk);
    if (keep && k < a.budget) {
      kept[k] = t;
      ns[k] = x;
    }
    eq += __popcll(be);
    place += __popcll(bk);
  });
}

// One block of the new cache, one head, K and V.  W: 4-byte words to a thread.
// 128 heads of 2048 tokens that stay, 128 wide: 47 us for 134 MB, 2.9 TB/s (26 us where the
// old cache is in the last-level cache): rows of 128 bytes from scattered places.  Four
// loads on their way instead of two: the same.
template <int W>
__global__ void __launch_bounds__(256) kv8_move_k(const EvictArgs a) {
  __shared__ int64_t at[128];
  __shared__ double ratio[2][128];  // of the scales; 1: the codes stay; -1: they are cleared
  __shared__ float top_s[4];
  const Cache &c = a.c, &o = a.to;
  const int blk = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int len = min(clampi(a.lengths[b], 0, c.cap), a.budget);
  const int p0 = blk << o.shift, nt = min(1 << o.shift, len - p0);
  if (nt <= 0) return;
  const int i = tid & 127, w = tid >> 7;  // K for half of the threads, V for the others
  float z = 0.f;
  if (i < nt) {
    const int t = clampi(a.kept[b * a.kp_seq + hk * a.kp_head + p0 + i], 0, c.cap - 1);
    if (w == 0) at[i] = b * c.st_seq + hk * c.st_head + t * c.st_token;
    z = (w ? c.vs : c.ks)[b * c.sc_seq + hk * c.sc_head + (t >> c.shift)];
  }
  float s = wave_max_dpp(z);
  if (__any(z != z)) s = NAN;
  if ((tid & 63) == 0) top_s[tid >> 6] = s;
  __syncthreads();
  s = max_nan(top_s[2 * w], top_s[2 * w + 1]);
  const bool live = s > 0.f && s < INFINITY;
  if (i < nt) ratio[w][i] = !live ? -1.0 : z == s ? 1.0 : (double)z / (double)s;
  if (i == 0) (w ? o.vs : o.ks)[b * o.sc_seq + hk * o.sc_head + blk] = s;
  __syncthreads();
  const int64_t to = b * o.st_seq + hk * o.st_head + p0 * o.st_token;
  const int parts = c.hs / (4 * W), n = nt * parts;
#pragma unroll 2
  for (int e = tid; e < 2 * n; e += 256) {
    const bool v = e >= n;
    const int f = v ? e - n : e, r = over(f, a.per), d = 4 * W * (f - r * parts);
    uint32_t x[W];
    __builtin_memcpy(x, __builtin_assume_aligned((v ? c.v : c.k) + at[r] + d, 4 * W), 4 * W);
    const double q = ratio[v][r];
    if (q != 1.0)
#pragma unroll
      for (int g = 0; g < W; g++) x[g] = q < 0.0 ? 0u : rescale4(x[g], q);
    __builtin_memcpy(__builtin_assume_aligned((v ? o.v : o.k) + to + r * o.st_token + d, 4 * W), x, 4 * W);
  }
}

// ------------------------------------------------------------- host side

// Element extent of one array of the cache, or -1 where rows would overlap.
int64_t code_span(const simp_rt_kv8 &c) {
  const int64_t in_head = c.st_head, in_tok = c.st_token, hs = c.head_size;
  int64_t span;
  auto step = [](int64_t n, int64_t st, int64_t inner, int64_t *out) {
    if (n > 1 && st < inner) return false;
    if (n > 1 && st > (INT64_MAX - inner) / (n - 1)) return false;
    *out = inner + (n > 1 ? (n - 1) * st : 0);
    return true;
  };
  int64_t a, s;
  if (step(c.capacity, in_tok, hs, &a) && step(c.n_kv_heads, in_head, a, &s)) span = s;
  else if (step(c.n_kv_heads, in_head, hs, &a) && step(c.capacity, in_tok, a, &s)) span = s;
  else return -1;
  return step(c.batch, c.st_seq, span, &s) ? s : -1;
}

int64_t scale_span(const simp_rt_kv8 &c) {
  const int64_t nb = cdiv(c.capacity, c.block);
  if (c.n_kv_heads > 1 && (c.sc_head < nb || c.sc_head > (INT64_MAX / 8 - nb) / (c.n_kv_heads - 1)))
    return -1;
  const int64_t in = nb + (c.n_kv_heads > 1 ? (c.n_kv_heads - 1) * c.sc_head : 0);
  if (c.batch > 1 && (c.sc_seq < in || c.sc_seq > (INT64_MAX / 8 - in) / (c.batch - 1))) return -1;
  return in + (c.batch > 1 ? (c.batch - 1) * c.sc_seq : 0);
}

// Whether K and V share codes or scales.  One may lie between the other's rows, heads or
// sequences, as the parts of one tensor do.
bool one_memory(const simp_rt_kv8 &c, int64_t codes, int64_t scales) {
  if (overlap(c.k, (size_t)codes, c.v, (size_t)codes)) {
    const Level seq{c.batch, c.st_seq}, head{c.n_kv_heads, c.st_head}, token{c.capacity, c.st_token}, d{c.head_size, 1};
    const bool heads_outside = c.n_kv_heads == 1 || c.capacity == 1 || c.st_head > c.st_token;
    const Level l[] = {seq, heads_outside ? head : token, heads_outside ? token : head, d};
    if (meet(l, 4, (int64_t)((uintptr_t)c.v - (uintptr_t)c.k))) return true;
  }
  if (overlap(c.k_scale, 4 * (size_t)scales, c.v_scale, 4 * (size_t)scales)) {
    const Level l[] = {{c.batch, c.sc_seq}, {c.n_kv_heads, c.sc_head}, {cdiv(c.capacity, c.block), 1}};
    if (meet(l, 3, (int64_t)((uintptr_t)c.v_scale - (uintptr_t)c.k_scale) / 4)) return true;
  }
  return false;
}

struct BoundCache {
  Operand k, v, ks, vs;
  Cache c;
  int64_t codes = 0, scales = 0;  // extents
  bool empty = false;
  int check(const simp_rt_kv8 *p, const char *fn, const char *name) {
    if (!p) return set_error(SIMP_RT_EINVAL, "%s: %s: null pointer", fn, name);
    if (p->batch < 0 || p->n_kv_heads < 0 || p->capacity < 0)
      return set_error(SIMP_RT_EINVAL, "%s: %s: negative size", fn, name);
    if (p->block != 16 && p->block != 32 && p->block != 64 && p->block != 128)
      return set_error(SIMP_RT_EINVAL, "%s: %s: block %lld is not 16, 32, 64 or 128", fn, name,
                       (long long)p->block);
    if (p->head_size < 16 || p->head_size > 256 || p->head_size % 4 != 0)
      return set_error(SIMP_RT_EUNSUPPORTED,
                       "%s: %s: head_size %lld is not a multiple of 4 in 16..256", fn, name,
                       (long long)p->head_size);
    if (p->st_token >= 1 << 24)
      return set_error(SIMP_RT_EUNSUPPORTED, "%s: %s: token stride of 2^24 or more", fn, name);
    if (p->batch > 32767 || p->n_kv_heads > 32767 || p->capacity > INT32_MAX - 4096)
      return set_error(SIMP_RT_EUNSUPPORTED, "%s: %s: batch or heads above 32767, or capacity above 2^31 - 4097",
                       fn, name);
    empty = p->batch == 0 || p->n_kv_heads == 0 || p->capacity == 0;
    if (empty) return SIMP_RT_OK;
    codes = code_span(*p);
    scales = scale_span(*p);
    if (codes < 0 || scales < 0)
      return set_error(SIMP_RT_EINVAL, "%s: %s: strides let rows overlap", fn, name);
    if (!p->k || !p->v || !p->k_scale || !p->v_scale)
      return set_error(SIMP_RT_EINVAL, "%s: %s: null pointer", fn, name);
    if (((uintptr_t)p->k | (uintptr_t)p->v | (uintptr_t)p->k_scale | (uintptr_t)p->v_scale |
         (uintptr_t)p->st_seq | (uintptr_t)p->st_head | (uintptr_t)p->st_token) & 3)
      return set_error(SIMP_RT_EINVAL, "%s: %s: rows and scales must start on 4-byte boundaries", fn, name);
    if (one_memory(*p, codes, scales))
      return set_error(SIMP_RT_EINVAL, "%s: %s: K and V share elements: the same memory", fn, name);
    return SIMP_RT_OK;
  }
  // Whether a byte range lies in one of the cache's arrays.
  bool shares(const simp_rt_kv8 *p, const void *q, size_t n) const {
    return overlap(q, n, p->k, (size_t)codes) || overlap(q, n, p->v, (size_t)codes) ||
           overlap(q, n, p->k_scale, 4 * (size_t)scales) ||
           overlap(q, n, p->v_scale, 4 * (size_t)scales);
  }
  int bind(const simp_rt_kv8 *p, Operand::Dir dir, int dev) {
    struct { Operand *o; const void *p; size_t n; const char *name; } a[] = {
        {&k, p->k, (size_t)codes, "cache k"}, {&v, p->v, (size_t)codes, "cache v"},
        {&ks, p->k_scale, 4 * (size_t)scales, "cache k_scale"},
        {&vs, p->v_scale, 4 * (size_t)scales, "cache v_scale"}};
    for (auto &x : a)  // no staging of whole caches
      if (int rc = bind_here(*x.o, x.p, x.n, dir, dev, x.name, false)) return rc;
    c.k = (int8_t *)k.dev(), c.v = (int8_t *)v.dev();
    c.ks = (float *)ks.dev(), c.vs = (float *)vs.dev();
    c.st_seq = p->st_seq, c.st_head = p->st_head, c.st_token = p->st_token;
    c.sc_seq = p->sc_seq, c.sc_head = p->sc_head;
    c.n = (int)p->batch, c.hk = (int)p->n_kv_heads, c.cap = (int)p->capacity, c.hs = (int)p->head_size;
    c.shift = __builtin_ctz((unsigned)p->block);
    return SIMP_RT_OK;
  }
};

// starts and lengths as every call takes them
int check_lists(const simp_rt_kv8 &c, const char *fn, const int32_t *starts, int64_t st_off,
                int64_t st_size, int64_t st_stride, const int32_t *lengths, int64_t len_off,
                int64_t len_size, int64_t len_stride, bool with_starts) {
  int rc;
  if (with_starts) {
    if ((rc = check_desc1("starts", starts, st_off, st_size, st_stride))) return rc;
    if (st_size != c.batch + 1)
      return set_error(SIMP_RT_EINVAL, "%s: starts must have batch + 1 entries", fn);
  }
  if ((rc = check_desc1("lengths", lengths, len_off, len_size, len_stride))) return rc;
  if (len_size != c.batch)
    return set_error(SIMP_RT_EINVAL, "%s: lengths must have batch entries", fn);
  return SIMP_RT_OK;
}

}  // namespace
}  // namespace simp

using namespace simp;

extern "C" {

int32_t simp_rt_kv8_append(
    const simp_rt_kv8 *cache, const float *k_alloc, const float *k, int64_t k_off, int64_t k_s0,
    int64_t k_s1, int64_t k_s2, int64_t k_st0, int64_t k_st1, int64_t k_st2, const float *v_alloc,
    const float *v, int64_t v_off, int64_t v_s0, int64_t v_s1, int64_t v_s2, int64_t v_st0,
    int64_t v_st1, int64_t v_st2, const int32_t *st_alloc, const int32_t *starts, int64_t st_off,
    int64_t st_size, int64_t st_stride, const int32_t *len_alloc, const int32_t *lengths,
    int64_t len_off, int64_t len_size, int64_t len_stride) {
  (void)k_alloc; (void)v_alloc; (void)st_alloc; (void)len_alloc;
  static const char *fn = "kv8_append";
  int rc;
  BoundCache bc;
  Desc3<const float> dk{k, k_off, {k_s0, k_s1, k_s2}, {k_st0, k_st1, k_st2}, 0};
  Desc3<const float> dv{v, v_off, {v_s0, v_s1, v_s2}, {v_st0, v_st1, v_st2}, 0};
  if ((rc = bc.check(cache, fn, "cache")) || (rc = dk.check("k")) || (rc = dv.check("v")) ||
      (rc = check_lists(*cache, fn, starts, st_off, st_size, st_stride, lengths, len_off, len_size,
                        len_stride, true)))
    return rc;
  if (!dk.is(k_s0, cache->n_kv_heads, cache->head_size) || !dv.is(k_s0, k_s1, k_s2))
    return set_error(SIMP_RT_EINVAL, "kv8_append: k and v must be [rows, n_kv_heads, head_size]");
  if (bc.empty || k_s0 == 0) return SIMP_RT_OK;
  if (bc.shares(cache, dk.data(), dk.bytes()) || bc.shares(cache, dv.data(), dv.bytes()) ||
      bc.shares(cache, starts + st_off, 4 * (size_t)st_size) ||
      bc.shares(cache, lengths + len_off, 4 * (size_t)len_size))
    return set_error(SIMP_RT_EINVAL, "kv8_append: rows or lists share memory with the cache");
  const int64_t slots = k_s0 / cache->block + 2 * cache->batch;
  if (k_s0 > INT32_MAX || slots * 1024 > UINT32_MAX)
    return set_error(SIMP_RT_EUNSUPPORTED, "kv8_append: more rows than the grid holds");
  const int dev = ensure_device();
  if (dev < 0) return dev;
  Operand ok, ov, os, ol;
  if ((rc = bc.bind(cache, Operand::kInOut, dev)) ||
      (rc = bind_here(ok, dk.data(), dk.bytes(), Operand::kIn, dev, "k")) ||
      (rc = bind_here(ov, dv.data(), dv.bytes(), Operand::kIn, dev, "v")) ||
      (rc = bind_here(os, starts + st_off, 4 * (size_t)st_size, Operand::kIn, dev, "starts")) ||
      (rc = bind_here(ol, lengths + len_off, 4 * (size_t)len_size, Operand::kIn, dev, "lengths")))
    return rc;
  const AppendArgs a{bc.c, (const float *)ok.dev(), (const float *)ov.dev(), (const int *)os.dev(),
                     (const int *)ol.dev(), dk.st[0], dk.st[1], dv.st[0], dv.st[1], (int)k_s0, per_of(bc.c.hs / 4)};
  const dim3 grid((unsigned)slots, (unsigned)bc.c.hk, 2);
  const bool vec = ((a.k_row | a.k_head | a.v_row | a.v_head) & 3) == 0 && (((uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0;
  const int64_t chunks = (int64_t)cache->block * bc.c.hs / 4;  // of a whole block
#define APPEND(N)                                                                              \
  do {                                                                                         \
    if (vec) hipLaunchKernelGGL((kv8_append_k<N, true>), grid, dim3(N), 0, cur_stream(), a);   \
    else hipLaunchKernelGGL((kv8_append_k<N, false>), grid, dim3(N), 0, cur_stream(), a);      \
  } while (0)
  if (chunks <= 64 * kAppendChunks) APPEND(64);
  else if (chunks <= 256 * kAppendChunks) APPEND(256);
  else APPEND(1024);
#undef APPEND
  Operand *ops[] = {&ok, &ov, &os, &ol};
  return finish(ops, 4);
}

int32_t simp_rt_kv8_read(
    const simp_rt_kv8 *cache, const int32_t *st_alloc, const int32_t *starts, int64_t st_off,
    int64_t st_size, int64_t st_stride, const int32_t *len_alloc, const int32_t *lengths,
    int64_t len_off, int64_t len_size, int64_t len_stride, float *k_alloc, float *k, int64_t k_off,
    int64_t k_s0, int64_t k_s1, int64_t k_s2, int64_t k_st0, int64_t k_st1, int64_t k_st2,
    float *v_alloc, float *v, int64_t v_off, int64_t v_s0, int64_t v_s1, int64_t v_s2,
    int64_t v_st0, int64_t v_st1, int64_t v_st2) {
  (void)k_alloc; (void)v_alloc; (void)st_alloc; (void)len_alloc;
  static const char *fn = "kv8_read";
  int rc;
  BoundCache bc;
  Desc3<float> dk{k, k_off, {k_s0, k_s1, k_s2}, {k_st0, k_st1, k_st2}, 0};
  Desc3<float> dv{v, v_off, {v_s0, v_s1, v_s2}, {v_st0, v_st1, v_st2}, 0};
  if ((rc = bc.check(cache, fn, "cache")) || (rc = dk.check("k")) || (rc = dv.check("v")) ||
      (rc = check_lists(*cache, fn, starts, st_off, st_size, st_stride, lengths, len_off, len_size,
                        len_stride, true)))
    return rc;
  if (!dk.is(k_s0, cache->n_kv_heads, cache->head_size) || !dv.is(k_s0, k_s1, k_s2))
    return set_error(SIMP_RT_EINVAL, "kv8_read: k and v must be [rows, n_kv_heads, head_size]");
  if (cache->batch == 0 || cache->n_kv_heads == 0 || k_s0 == 0) return SIMP_RT_OK;
  if (cdiv(k_s0, kReadRows) * 256 > UINT32_MAX)
    return set_error(SIMP_RT_EUNSUPPORTED, "kv8_read: more rows than the grid holds");
  if (bc.empty) return set_error(SIMP_RT_EINVAL, "kv8_read: the cache has no capacity");
  if (bc.shares(cache, dk.data(), dk.bytes()) || bc.shares(cache, dv.data(), dv.bytes()))
    return set_error(SIMP_RT_EINVAL, "kv8_read: rows share memory with the cache");
  if (share(dk, dv) || overlap(dk.data(), dk.bytes(), starts + st_off, 4 * (size_t)st_size) ||
      overlap(dv.data(), dv.bytes(), starts + st_off, 4 * (size_t)st_size) ||
      overlap(dk.data(), dk.bytes(), lengths + len_off, 4 * (size_t)len_size) ||
      overlap(dv.data(), dv.bytes(), lengths + len_off, 4 * (size_t)len_size))
    return set_error(SIMP_RT_EINVAL, "kv8_read: k or v shares memory with another operand");
  const int dev = ensure_device();
  if (dev < 0) return dev;
  Operand ok, ov, os, ol;
  if ((rc = bc.bind(cache, Operand::kIn, dev)) ||
      (rc = bind_here(ok, dk.data(), dk.bytes(), Operand::kOut, dev, "k")) ||
      (rc = bind_here(ov, dv.data(), dv.bytes(), Operand::kOut, dev, "v")) ||
      (rc = bind_here(os, starts + st_off, 4 * (size_t)st_size, Operand::kIn, dev, "starts")) ||
      (rc = bind_here(ol, lengths + len_off, 4 * (size_t)len_size, Operand::kIn, dev, "lengths")))
    return rc;
  dk.rows_of(ok), dv.rows_of(ov);  // they may lie between each other's
  const ReadArgs a{bc.c, (const int *)os.dev(), (const int *)ol.dev(), (float *)ok.dev(),
                   (float *)ov.dev(), dk.st[0], dk.st[1], dv.st[0], dv.st[1], (int)k_s0};
  const dim3 grid((unsigned)cdiv(k_s0, kReadRows), (unsigned)bc.c.hk);
  if (((a.k_row | a.k_head | a.v_row | a.v_head) & 3) == 0 && (((uintptr_t)a.k | (uintptr_t)a.v) & 15) == 0)
    hipLaunchKernelGGL(kv8_read_k<true>, grid, dim3(256), 0, cur_stream(), a);
  else
    hipLaunchKernelGGL(kv8_read_k<false>, grid, dim3(256), 0, cur_stream(), a);
  Operand *ops[] = {&ok, &ov, &os, &ol};
  return finish(ops, 4);
}

int32_t simp_rt_kv8_attention(
    const simp_rt_kv8 *cache, const float *q_alloc, const float *q, int64_t q_off, int64_t q_s0,
    int64_t q_s1, int64_t q_s2, int64_t q_st0, int64_t q_st1, int64_t q_st2,
    const int32_t *len_alloc, const int32_t *lengths, int64_t len_off, int64_t len_size,
    int64_t len_stride, float *out_alloc, float *out, int64_t out_off, int64_t out_s0,
    int64_t out_s1, int64_t out_s2, int64_t out_st0, int64_t out_st1, int64_t out_st2,
    const float *si_alloc, const float *seen_in, int64_t si_off, int64_t si_s0, int64_t si_s1,
    int64_t si_s2, int64_t si_st0, int64_t si_st1, int64_t si_st2, float *so_alloc,
    float *seen_out, int64_t so_off, int64_t so_s0, int64_t so_s1, int64_t so_s2, int64_t so_st0,
    int64_t so_st1, int64_t so_st2, double scale) {
  (void)q_alloc; (void)len_alloc; (void)out_alloc; (void)si_alloc; (void)so_alloc;
  static const char *fn = "kv8_attention";
  int rc;
  BoundCache bc;
  Desc3<const float> dq{q, q_off, {q_s0, q_s1, q_s2}, {q_st0, q_st1, q_st2}, 0};
  Desc3<float> dout{out, out_off, {out_s0, out_s1, out_s2}, {out_st0, out_st1, out_st2}, 0};
  Desc3<const float> dsi{seen_in, si_off, {si_s0, si_s1, si_s2}, {si_st0, si_st1, si_st2}, 0};
  Desc3<float> dso{seen_out, so_off, {so_s0, so_s1, so_s2}, {so_st0, so_st1, so_st2}, 0};
  const bool with = seen_in || seen_out;
  if ((rc = bc.check(cache, fn, "cache")) || (rc = dq.check("q")) || (rc = dout.check("out")) ||
      (rc = check_lists(*cache, fn, nullptr, 0, 0, 0, lengths, len_off, len_size, len_stride, false)))
    return rc;
  if (with && ((rc = dsi.check("seen_in")) || (rc = dso.check("seen_out")))) return rc;
  if (!dq.is(cache->batch, q_s1, cache->head_size) || !dout.is(q_s0, q_s1, q_s2))
    return set_error(SIMP_RT_EINVAL, "kv8_attention: q and out must be [batch, heads, head_size]");
  if (q_s0 == 0 || q_s1 == 0) return SIMP_RT_OK;
  if (cache->n_kv_heads < 1 || q_s1 % cache->n_kv_heads != 0)
    return set_error(SIMP_RT_EINVAL, "kv8_attention: %lld heads are no multiple of %lld kv heads",
                     (long long)q_s1, (long long)cache->n_kv_heads);
  if (bc.empty) return set_error(SIMP_RT_EINVAL, "kv8_attention: the cache has no capacity");
  if (with && (!dsi.is(cache->batch, cache->n_kv_heads, cache->capacity) || !dso.is(si_s0, si_s1, si_s2)))
    return set_error(SIMP_RT_EINVAL, "kv8_attention: seen_in and seen_out must be [batch, n_kv_heads, capacity]");
  if (!scale_fits(scale)) return set_error(SIMP_RT_EINVAL, "kv8_attention: scale must be finite, also in fp32 and times log2(e)");
  if (q_s1 > 32767 || q_s1 / cache->n_kv_heads > 4096)
    return set_error(SIMP_RT_EUNSUPPORTED, "kv8_attention: heads above 32767, or 4096 to a kv head");
  const bool in_place = with && dsi.data() == dso.data() && dsi.st[0] == dso.st[0] && dsi.st[1] == dso.st[1];
  const auto with_lengths = [&](const void *p, size_t n) { return overlap(p, n, lengths + len_off, 4 * (size_t)len_size); };
  if (overlap(dout.data(), dout.bytes(), dq.data(), dq.bytes()) ||
      bc.shares(cache, dout.data(), dout.bytes()) || with_lengths(dout.data(), dout.bytes()) ||
      (with && with_lengths(dso.data(), dso.bytes())) ||
      (with && bc.shares(cache, dso.data(), dso.bytes())) ||
      (with && (overlap(dout.data(), dout.bytes(), dsi.data(), dsi.bytes()) ||
                overlap(dout.data(), dout.bytes(), dso.data(), dso.bytes()) ||
                overlap(dso.data(), dso.bytes(), dq.data(), dq.bytes()) ||
                (!in_place && overlap(dsi.data(), dsi.bytes(), dso.data(), dso.bytes())))))
    return set_error(SIMP_RT_EINVAL, "kv8_attention: an output shares memory with another operand");
  const int dev = ensure_device();
  if (dev < 0) return dev;
  Operand oq, ol, oo, osi, oso;
  if ((rc = bc.bind(cache, Operand::kIn, dev)) ||
      (rc = bind_here(oq, dq.data(), dq.bytes(), Operand::kIn, dev, "q")) ||
      (rc = bind_here(ol, lengths + len_off, 4 * (size_t)len_size, Operand::kIn, dev, "lengths")) ||
      (rc = bind_here(oo, dout.data(), dout.bytes(), Operand::kOut, dev, "out")) ||
      (with && ((rc = bind_here(osi, dsi.data(), dsi.bytes(), Operand::kIn, dev, "seen_in")) ||
                (rc = bind_here(oso, dso.data(), dso.bytes(), Operand::kOut, dev, "seen_out")))))
    return rc;
  AttnArgs a{};
  a.c = bc.c;
  a.q = (const float *)oq.dev();
  a.lengths = (const int *)ol.dev();
  a.out = (float *)oo.dev();
  a.seen_in = (const float *)osi.dev();
  a.seen_out = (float *)oso.dev();
  a.q_seq = dq.st[0], a.q_head = dq.st[1], a.o_seq = dout.st[0], a.o_head = dout.st[1];
  a.si_seq = dsi.st[0], a.si_head = dsi.st[1], a.so_seq = dso.st[0], a.so_head = dso.st[1];
  a.heads = (int)q_s1, a.group = (int)(q_s1 / cache->n_kv_heads);
  a.scale = (float)(scale * 1.4426950408889634);
  hipStream_t st = cur_stream();
  // Pieces for two blocks a CU, three where four waves fit a SIMD: what a block does once
  // (lengths, q, its rows joined and written) costs it as much as several tiles.  16
  // ragged sequences of up to 4096, 128 wide: 19.4 us with 256 pieces, 15.9 with 512, 16.2
  // with 768, 18.2 with 1024; 64 of them, 64 wide: 49, 37, 33.6 and 34.7 us; 131072 tokens of
  // one: 58.5, 58.8, 62 and 58.
  // A quad of lanes to a head up to four of them; else 16, or the 8 whose rows fit 64 KB
  // of LDS.
  a.width = a.group <= 4 ? 4 : bc.c.hs > 192 ? 8 : 16;
  a.sets = (int)cdiv(a.group, a.width);
  const int64_t units = (int64_t)bc.c.n * bc.c.hk * a.sets, most = units * cdiv(bc.c.cap, kRound);
  a.blocks = num_cus() * (bc.c.hs <= 64 ? 3 : 2);
  const int64_t pieces = std::min(units + a.blocks, most);  // every unit may have one that is not full
  if (most > INT32_MAX - a.blocks || pieces > UINT32_MAX / 256)
    return set_error(SIMP_RT_EUNSUPPORTED, "kv8_attention: more heads and tokens than the kernels count");
  const size_t rows = (size_t)q_s0 * (size_t)q_s1, parts = (size_t)pieces * (size_t)a.width;
  Workspace ws;
  float *p = nullptr;
  a.score_row = cdiv(bc.c.cap, 64) * 64;
  const size_t scores = with ? rows * (size_t)a.score_row : 0;
  if ((rc = ws.get(st, 4 * (scores + parts * (size_t)(bc.c.hs + 2) + (size_t)bc.c.n + 2), (void **)&p, 8))) return rc;
  a.scores = with ? p : nullptr;
  a.part = p + scores;
  a.stat = (float2 *)(a.part + parts * (size_t)bc.c.hs);
  a.starts = (int *)(a.stat + parts);
  const size_t cols = (size_t)std::min(a.group, a.width);
  const unsigned lds = (unsigned)(4 * 4 * cols * ((size_t)bc.c.hs + 2));
  if (bc.c.n > 64) hipLaunchKernelGGL(kv8_plan_k, dim3(1), dim3(1024), 0, st, a);
  const dim3 grid((unsigned)pieces);
#define ATTN(NC)                                                                      \
  do {                                                                                \
    if (a.group <= 4) hipLaunchKernelGGL((kv8_attn_k<NC, true>), grid, dim3(256), lds, st, a); \
    else hipLaunchKernelGGL((kv8_attn_k<NC, false>), grid, dim3(256), lds, st, a);    \
  } while (0)
  if (bc.c.hs <= 64) ATTN(1);
  else if (bc.c.hs <= 128) ATTN(2);
  else if (bc.c.hs <= 192) ATTN(3);
  else ATTN(4);
#undef ATTN
  // The accumulated weights 512 tokens to a block, and twice as many where that would make
  // more than four blocks a CU: 16 sequences of up to 4096 tokens (1024 blocks) 4.8 us
  // against 5.4, 131072 tokens of one (2048) 10.1 against 8.0.
  const int64_t tiles = with ? cdiv(bc.c.cap, 512) : 0;
  const bool wide = tiles * bc.c.hk * bc.c.n > 4 * num_cus();
  const dim3 joins((unsigned)(a.group + (wide ? cdiv(tiles, 2) : tiles)), (unsigned)bc.c.hk, (unsigned)bc.c.n);
  const unsigned sums = (unsigned)(4 * std::max<int64_t>(std::min<int64_t>(a.blocks, cdiv(bc.c.cap, kRound)), 2 * a.group));
  if (wide) hipLaunchKernelGGL(kv8_join_k<1024>, joins, dim3(256), sums, st, a);
  else hipLaunchKernelGGL(kv8_join_k<512>, joins, dim3(256), sums, st, a);
  Operand *ops[] = {&oq, &ol, &oo, &osi, &oso};
  return finish(ops, with ? 5 : 3);
}

int32_t simp_rt_kv8_evict(
    const simp_rt_kv8 *cache, const simp_rt_kv8 *to, const int32_t *len_alloc,
    const int32_t *lengths, int64_t len_off, int64_t len_size, int64_t len_stride,
    const float *se_alloc, const float *seen, int64_t se_off, int64_t se_s0, int64_t se_s1,
    int64_t se_s2, int64_t se_st0, int64_t se_st1, int64_t se_st2, float *ns_alloc,
    float *new_seen, int64_t ns_off, int64_t ns_s0, int64_t ns_s1, int64_t ns_s2, int64_t ns_st0,
    int64_t ns_st1, int64_t ns_st2, int32_t *kept_alloc, int32_t *kept, int64_t kept_off,
    int64_t kept_s0, int64_t kept_s1, int64_t kept_s2, int64_t kept_st0, int64_t kept_st1,
    int64_t kept_st2, int64_t budget, int64_t recent) {
  (void)len_alloc; (void)se_alloc; (void)ns_alloc; (void)kept_alloc;
  static const char *fn = "kv8_evict";
  int rc;
  BoundCache bc, bt;
  Desc3<const float> ds{seen, se_off, {se_s0, se_s1, se_s2}, {se_st0, se_st1, se_st2}, 0};
  Desc3<float> dn{new_seen, ns_off, {ns_s0, ns_s1, ns_s2}, {ns_st0, ns_st1, ns_st2}, 0};
  Desc3<int32_t> dp{kept, kept_off, {kept_s0, kept_s1, kept_s2}, {kept_st0, kept_st1, kept_st2}, 0};
  if ((rc = bc.check(cache, fn, "cache")) || (rc = bt.check(to, fn, "to")) ||
      (rc = ds.check("seen")) || (rc = dn.check("new_seen")) || (rc = dp.check("kept")) ||
      (rc = check_lists(*cache, fn, nullptr, 0, 0, 0, lengths, len_off, len_size, len_stride, false)))
    return rc;
  if (to->batch != cache->batch || to->n_kv_heads != cache->n_kv_heads ||
      to->head_size != cache->head_size || to->block != cache->block)
    return set_error(SIMP_RT_EINVAL, "kv8_evict: the caches differ in batch, heads, head_size or block");
  if (budget < 0 || budget > to->capacity || recent < 0 || recent > budget)
    return set_error(SIMP_RT_EINVAL, "kv8_evict: budget %lld (capacity %lld), recent %lld: "
                     "0 <= recent <= budget <= the new cache's capacity is wanted", (long long)budget,
                     (long long)to->capacity, (long long)recent);
  if (!ds.is(cache->batch, cache->n_kv_heads, cache->capacity) ||
      !dp.is(cache->batch, cache->n_kv_heads, budget) || ns_s0 != cache->batch ||
      ns_s1 != cache->n_kv_heads || ns_s2 < budget)
    return set_error(SIMP_RT_EINVAL, "kv8_evict: seen must be [batch, n_kv_heads, capacity], new_seen "
                     "[batch, n_kv_heads, >= budget], kept [batch, n_kv_heads, budget]");
  if (budget == 0 || cache->batch == 0 || cache->n_kv_heads == 0) return SIMP_RT_OK;
  if (bc.empty) return set_error(SIMP_RT_EINVAL, "kv8_evict: the cache has no capacity");
  const struct { const void *p; size_t n; } r[] = {
      {to->k, (size_t)bt.codes}, {to->v, (size_t)bt.codes}, {to->k_scale, 4 * (size_t)bt.scales},
      {to->v_scale, 4 * (size_t)bt.scales}, {dn.data(), dn.bytes()}, {dp.data(), dp.bytes()},
      {cache->k, (size_t)bc.codes}, {cache->v, (size_t)bc.codes},
      {cache->k_scale, 4 * (size_t)bc.scales}, {cache->v_scale, 4 * (size_t)bc.scales},
      {ds.data(), ds.bytes()}, {lengths + len_off, 4 * (size_t)len_size}};
  for (int i = 0; i < 6; i++)
    for (int j = i + 1; j < 12; j++) {
      if (i < 4 && j < 4) continue;  // the new cache's own arrays may be interleaved
      if (overlap(r[i].p, r[i].n, r[j].p, r[j].n))
        return set_error(SIMP_RT_EINVAL, "kv8_evict: an output shares memory with another operand");
    }
  const int dev = ensure_device();
  if (dev < 0) return dev;
  Operand ol, os, on, op;
  if ((rc = bc.bind(cache, Operand::kIn, dev)) || (rc = bt.bind(to, Operand::kOut, dev)) ||
      (rc = bind_here(ol, lengths + len_off, 4 * (size_t)len_size, Operand::kIn, dev, "lengths")) ||
      (rc = bind_here(os, ds.data(), ds.bytes(), Operand::kIn, dev, "seen")) ||
      (rc = bind_here(on, dn.data(), dn.bytes(), Operand::kOut, dev, "new_seen")) ||
      (rc = bind_here(op, dp.data(), dp.bytes(), Operand::kOut, dev, "kept")))
    return rc;
  EvictArgs a{bc.c, bt.c, (const int *)ol.dev(), (const float *)os.dev(), (float *)on.dev(),
                    (int *)op.dev(), ds.st[0], ds.st[1], dn.st[0], dn.st[1], dp.st[0], dp.st[1],
                    (int)budget, (int)recent, 0};
  hipStream_t st = cur_stream();
  hipLaunchKernelGGL(kv8_select_k, dim3((unsigned)bc.c.hk, (unsigned)bc.c.n), dim3(1024), 0, st, a);
  const dim3 grid((unsigned)cdiv(budget, to->block), (unsigned)bc.c.hk, (unsigned)bc.c.n);
  auto wide = [](const Cache &c) {
    return ((c.hs | c.st_seq | c.st_head | c.st_token | (int64_t)(uintptr_t)c.k | (int64_t)(uintptr_t)c.v) & 15) == 0;
  };
  const bool quads = wide(bc.c) && wide(bt.c);
  a.per = per_of(bc.c.hs / (quads ? 16 : 4));
  if (quads) hipLaunchKernelGGL(kv8_move_k<4>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(kv8_move_k<1>, grid, dim3(256), 0, st, a);
  Operand *ops[] = {&ol, &os, &on, &op};
  return finish(ops, 4);
}

}  // extern "C"
