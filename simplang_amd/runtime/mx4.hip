// mx4.hip -- microscaled 4-bit floating point (MXFP4): quantisation, products and the
// gated half of a feed-forward block.
//
// A value is an E2M1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) times a power of two
// that 32 elements of a row share (OCP Microscaling Formats specification 1.0).
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies such operands as they are: lane l of a
// wave holds the 32 codes (16 bytes) of block l / 16 of row l % 16, and their scale in a
// byte of another register, so that an MX block is what one lane brings and nothing is
// unpacked.  Checked on the device: products are exact, and the sum of 128 of them and
// the accumulator is rounded to nearest in fp32, subnormals kept (two blocks' sums that
// lie 2^24 apart are rounded where they meet); a scale byte of 255 makes the sum NaN,
// also where the codes are 0.
#include <algorithm>
#include <type_traits>

#include "rt_device.h"
#include "rt_internal.h"
#include "serve_args.h"

namespace simp {
namespace {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
// Loads and stores at any address their element allows (the type says so; the
// compiler picks the instructions).
typedef uint32_t u4any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u1any __attribute__((aligned(1)));
typedef uint16_t u2any __attribute__((aligned(1)));
typedef float f4any __attribute__((ext_vector_type(4), aligned(4)));

// Sixteen bytes at any address.  `shift` (uniform): aligned dwords put together, which may
// begin up to three bytes ahead of p; a load that the memory path splits takes longer.
__device__ __forceinline__ uint4 load16(const uint8_t *p, bool shift = false) {
  if (shift) {
    const uint32_t sh = (uintptr_t)p & 3;
    const u4any u = *(const u4any *)__builtin_assume_aligned(p - sh, 4);
    const uint32_t w = *(const u1any *)(p + 12);
    return make_uint4(__builtin_amdgcn_alignbyte(u.y, u.x, sh), __builtin_amdgcn_alignbyte(u.z, u.y, sh),
                      __builtin_amdgcn_alignbyte(u.w, u.z, sh), w);
  }
  const u4any v = *(const u4any *)p;
  return make_uint4(v.x, v.y, v.z, v.w);
}

__device__ __forceinline__ uint32_t max_dpp8(uint32_t v) {  // over lanes 8i .. 8i+7
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kDppXor1, 0xF, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kDppXor2, 0xF, 0xF, false));
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kDppHalfMirror, 0xF, 0xF, false));
}

// 2^(s - 127) in fp32 (255: infinity)
__device__ __forceinline__ float scale_of(uint32_t s) {
  return __uint_as_float(s ? s << 23 : 0x00400000u);
}

// Row and column block of the i-th 32-element block (or 16-byte piece) of the rows, i counted from
// the workgroup's first, which is below 2^31 (the callers hold the grid to it), as is per_row.
struct BlockAt {
  int64_t row0;
  uint32_t rem, per;
  __device__ BlockAt(int64_t first, int64_t per_row) {
    per = (uint32_t)per_row;
    row0 = (uint32_t)first / per;
    rem = (uint32_t)(first - row0 * per_row);
  }
  __device__ void get(uint32_t i, int64_t &row, int64_t &blk) const {
    const uint32_t q = (rem + i) / per;
    row = row0 + q;
    blk = rem + i - q * per;
  }
};

// Eight lanes to a block, four elements each, so that a wave's loads and stores of values are
// 1 KB in lane order; a thread takes RUN blocks, their loads together.  STREAM: values are
// taken and left past the caches (they lie on 16 bytes).  8192 x 8192: 59 us (5.1 TB/s) and
// back 44 us (6.9; a copy reaches 4.9); with eight elements to a lane, 32 bytes apart, 75
// and 78.  RUN: 1 to 2^15 blocks, where few leave CUs idle (in a graph 1 x 3200: 2.3 us and back
// 2.5, with 4 3.2 and 3.1; 1024 x 992: 2.8 and 3.1, with 4 3.7 and 3.9), above it 4, which the
// largest are better with (4096 x 4096 back: 12.4 us, with 1 13.6; 8192 x 8192 44, with 1 68, not past
// the caches).  Just above 2^15 it costs a microsecond (717 x 1533: 4.1 and 4.1, with 1 3.1 and 3.4).
template <int RUN, bool STREAM>
__global__ void __launch_bounds__(256)
    quantize_mx4_k(const float *__restrict__ x, int64_t ldx, uint8_t *__restrict__ codes,
                   int64_t ldc, uint8_t *__restrict__ scales, int64_t lds, int64_t cols,
                   int64_t per_row, int64_t blocks) {
  const int64_t first = (int64_t)blockIdx.x * (32 * RUN);
  const BlockAt at(first, per_row);
  const int lane8 = threadIdx.x & 7;
  int64_t row[RUN], blk[RUN];
  v4f v[RUN];
#pragma unroll
  for (int u = 0; u < RUN; u++) {
    const uint32_t i = u * 32 + (threadIdx.x >> 3);
    at.get(i, row[u], blk[u]);
    const int64_t c0 = 32 * blk[u] + 4 * lane8;
    const float *p = x + row[u] * ldx + c0;
    v[u] = v4f{0.f, 0.f, 0.f, 0.f};
    if (first + i >= blocks) continue;  // the eight lanes of a block together
    if (c0 + 4 <= cols) {
      if constexpr (STREAM) v[u] = __builtin_nontemporal_load((const v4f *)p);
      else v[u] = *(const f4any *)p;
    } else {
#pragma unroll
      for (int e = 0; e < 3; e++)
        if (c0 + e < cols) v[u][e] = p[e];
    }
  }
#pragma unroll
  for (int u = 0; u < RUN; u++) {
    if (first + u * 32 + (threadIdx.x >> 3) >= blocks) break;
    const int64_t c0 = 32 * blk[u] + 4 * lane8;
    uint32_t top = 0;  // sizes compare as whole numbers, NaN above infinity
#pragma unroll
    for (int e = 0; e < 4; e++) top = max(top, __float_as_uint(v[u][e]) & 0x7FFFFFFFu);
    top = max_dpp8(top);
    const bool bad = top >= 0x7F800000u;
    const uint32_t ex = top >> 23, s = ex > 2 ? ex - 2 : 0;
    const float unit = scale_of(s);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[u][0], v[u][1], unit, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[u][2], v[u][3], unit, 1);
    if (bad) c = 0;
    uint8_t *o = codes + row[u] * ldc + (c0 >> 1);
    if (c0 + 4 <= cols) {
      *(u2any *)o = (uint16_t)c;
    } else {
#pragma unroll
      for (int e = 0; e < 2; e++)
        if (c0 + 2 * e < cols) o[e] = (uint8_t)(c >> (8 * e));
    }
    if (lane8 == 0) scales[row[u] * lds + blk[u]] = bad ? 255 : (uint8_t)s;
  }
}

template <int RUN, bool STREAM>
__global__ void __launch_bounds__(256)
    dequantize_mx4_k(const uint8_t *__restrict__ codes, int64_t ldc,
                     const uint8_t *__restrict__ scales, int64_t lds, float *__restrict__ out,
                     int64_t ldo, int64_t cols, int64_t per_row, int64_t blocks) {
  const int64_t first = (int64_t)blockIdx.x * (32 * RUN);
  const BlockAt at(first, per_row);
  const int lane8 = threadIdx.x & 7;
  int64_t row[RUN], blk[RUN];
  uint32_t c[RUN], s[RUN];
#pragma unroll
  for (int u = 0; u < RUN; u++) {
    const uint32_t i = u * 32 + (threadIdx.x >> 3);
    at.get(i, row[u], blk[u]);
    const int64_t c0 = 32 * blk[u] + 4 * lane8;
    const uint8_t *p = codes + row[u] * ldc + (c0 >> 1);
    c[u] = s[u] = 0;
    if (first + i >= blocks || c0 >= cols) continue;
    if (c0 + 4 <= cols) {
      c[u] = *(const u2any *)p;
    } else {
      c[u] = p[0];
      if (c0 + 2 < cols) c[u] |= (uint32_t)p[1] << 8;
    }
    s[u] = scales[row[u] * lds + blk[u]];
  }
#pragma unroll
  for (int u = 0; u < RUN; u++) {
    const int64_t c0 = 32 * blk[u] + 4 * lane8;
    if (first + u * 32 + (threadIdx.x >> 3) >= blocks || c0 >= cols) continue;
    const float unit = scale_of(s[u]);
    const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], unit, 0),
              b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], unit, 1);
    v4f v = {a[0], a[1], b[0], b[1]};
    if (s[u] == 255) {
      const float nan = __uint_as_float(0x7FC00000u);
      v = v4f{nan, nan, nan, nan};
    }
    float *o = out + row[u] * ldo + c0;
    if (c0 + 4 <= cols) {
      if constexpr (STREAM) __builtin_nontemporal_store(v, (v4f *)o);
      else *(f4any *)o = v;
    } else {
#pragma unroll
      for (int e = 0; e < 3; e++)
        if (c0 + e < cols) o[e] = v[e];
    }
  }
}

// ------------------------------------------------------------------ products

struct Mx4Args {
  const uint8_t *a, *as, *b[2], *bs[2];  // codes and scales of A, and of B or W1 and W3
  int64_t lda, ldas, ldb[2], ldbs[2];
  float *out;
  int64_t ldo;
  int M, N, kb;  // kb: code bytes of a row
  bool shift;    // rows of scales not on 4 bytes, but the arrays' first bytes are
  bool shift_codes;  // the same for rows of codes, and no array's first byte is in the way
};

__device__ __forceinline__ v4f mfma_mx4(uint4 a, uint32_t sa, uint4 b, uint32_t sb, v4f c) {
  const v8i x = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0},
            y = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, 0, (int)sa, 0, (int)sb);
}

// silu(g) * u = g / (1 + exp(-g)) * u within 8 half units: with t = fl(x log2(e)), exp(x) is
// 2^t (1 + x - t ln 2), which leaves the rounding of t (it would count |x| times) out.  From
// x = 88.7228394 on, the first for which t reaches 128, exp is infinite and silu 0.  Quarters of
// g and of the divisor: the reciprocal of a number above 2^126 is subnormal, and comes out as 0.
// A gate costs what its instructions do, 64 to a lane and tile with the matrix cores idle:
// 4096 x 2048 x 8192 takes 87 us in the 256 x 256 tiles, with expf and a division 98, with a
// Newton step for the reciprocal 90 (error in the 2-norm 5.25e-8, 4.95e-8, 5.20e-8).
__device__ __forceinline__ float swiglu(float g, float u) {
  const float x = __builtin_amdgcn_fmed3f(-g, -200.f, 88.7228394f), t = x * 1.44269504f;
  const float low = fmaf(-t, -1.90465421e-9f, fmaf(-t, 0.693147182f, x));  // ln 2 in two parts
  const float p = __builtin_amdgcn_exp2f(t), e = fmaf(p, low, p);
  return 0.25f * g * __builtin_amdgcn_rcpf(fmaf(e, 0.25f, 0.25f)) * u;
}

// Exchanges registers and lanes: of n = 2 or 4 neighbouring lanes, lane t gets in y[s] what
// lane s has in x[t].  A fragment of the products leaves a lane four columns of one row, 64
// bytes for each of 16 rows to a store; of n fragments side by side this makes n stores of
// 64 n bytes for each of 16 / n rows, whole lines, which the memory takes in half the time.
template <int N>
__device__ __forceinline__ void lane_transpose(v4f (&x)[N]) {
  const int t = threadIdx.x;
  auto swap = [&](v4f &a, v4f &b, auto ctrl, bool odd) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const float u = dpp_mov<decltype(ctrl)::value>(b[e]), v = dpp_mov<decltype(ctrl)::value>(a[e]);
      a[e] = odd ? u : a[e];
      b[e] = odd ? b[e] : v;
    }
  };
#pragma unroll
  for (int i = 0; i < N; i += 2) swap(x[i], x[i + 1], std::integral_constant<int, kDppXor1>{}, t & 1);
  if constexpr (N == 4) {
    swap(x[0], x[2], std::integral_constant<int, kDppXor2>{}, t & 2);
    swap(x[1], x[3], std::integral_constant<int, kDppXor2>{}, t & 2);
  }
}

// 16 bytes of a row of kb from byte k on, zeros behind its end: with fewer left, the row's last
// 16 shifted down.  In two parts, so that many loads can be on their way: what to load, ...
__device__ __forceinline__ uint4 row_load(const uint8_t *row, int k, int kb) {
  if (kb >= 16) return load16(row + min(k, kb - 16));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 15; i++)
    if (k + i < kb) w[i >> 2] |= (uint32_t)row[k + i] << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// ... and what to make of it.
__device__ __forceinline__ uint4 shift_down(uint4 v, int bytes) {  // 0 to 16
  uint64_t lo = v.x | (uint64_t)v.y << 32, hi = v.z | (uint64_t)v.w << 32;
  if (bytes >= 8) lo = bytes < 16 ? hi >> (8 * (bytes - 8)) : 0, hi = 0;
  else if (bytes > 0) lo = lo >> (8 * bytes) | hi << (64 - 8 * bytes), hi >>= 8 * bytes;
  return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}
__device__ __forceinline__ uint4 row_shift(uint4 v, int k, int kb) {
  return kb >= 16 ? shift_down(v, min(max(k - kb + 16, 0), 16)) : v;
}

// 16 columns of each matrix and all 16 MT rows to a block, whose waves split K: a wave
// takes every byte of its rows' piece once, straight from memory into the lanes that
// feed the matrix instruction (16 rows of 64 bytes, and a byte of scales to a lane), and
// the waves' sums meet in LDS, in the order of K.  SHIFT: rows of scales (1), of codes too (2),
// that are not on 4 bytes are read as aligned dwords (16 x 8641 x 3200: 9.1 us, 14.6 as
// they lie; 16 x 8640 x 3200, where only the scales are not, 6.6).  Memory bounds it, 1 x 3200 x 32000:
// 10.0 us, 5.4 TB/s of weights that lie in the last cache; 16 x 3200 x 8640 gated 7.6.
constexpr int skinny_waves(int MT, int MATS) { return MT * MATS >= 4 ? 8 : 16; }  // of a block at most
template <int MT, int MATS, int SHIFT>
__global__ void __launch_bounds__(64 * skinny_waves(MT, MATS)) mx4_skinny_k(const Mx4Args a, int span, int blocks_n) {
  constexpr int T = MATS * MT;
  constexpr int U = MT == 4 ? 2 : 4;
  extern __shared__ v4f part[];  // [waves][T][64]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int r = lane & 15, q = lane >> 4;
  const int bm = blockIdx.x / blocks_n;
  const int n0 = 16 * (blockIdx.x - bm * blocks_n), m0 = 16 * MT * bm;
  const uint8_t *ap[MT], *as[MT], *bp[MATS], *bs[MATS];
  bool in[MT];  // rows behind the last are not asked for
#pragma unroll
  for (int i = 0; i < MT; i++) {
    in[i] = m0 + 16 * i + r < a.M;
    const int64_t m = min(m0 + 16 * i + r, a.M - 1);
    ap[i] = a.a + m * a.lda, as[i] = a.as + m * a.ldas;
  }
#pragma unroll
  for (int t = 0; t < MATS; t++) {
    const int64_t n = min(n0 + r, a.N - 1);
    bp[t] = a.b[t] + n * a.ldb[t], bs[t] = a.bs[t] + n * a.ldbs[t];
  }
  v4f acc[MATS][MT];
#pragma unroll
  for (int t = 0; t < MATS; t++)
#pragma unroll
    for (int i = 0; i < MT; i++) acc[t][i] = v4f{0.f, 0.f, 0.f, 0.f};
  struct Step {
    uint4 a[MT], b[MATS];
    uint32_t as[MT], bs[MATS];
  };
  auto run = [&](const Step &s) {
#pragma unroll
    for (int t = 0; t < MATS; t++)
#pragma unroll
      for (int i = 0; i < MT; i++) acc[t][i] = mfma_mx4(s.b[t], s.bs[t], s.a[i], s.as[i], acc[t][i]);
  };
  // Four steps: a lane's four scale bytes come out of 16 of its row.  What bounds the loop is
  // the path from the caches, 64 bytes a cycle and a row to a cycle: a byte of scales for
  // each fragment and step would cost as much as the codes.  `edge`: rows may end in them.
  const int nb = (a.kb + 15) >> 4;
  auto four = [&](int s, int end, auto edge) {
    constexpr int E = decltype(edge)::value;  // 2: rows shorter than 16 bytes
    auto load = [&](const uint8_t *row, int k, int size) {
      if constexpr (E == 2) return row_load(row, k, size);
      else return load16(row + (E ? min(k, size - 16) : k), SHIFT == 2);
    };
    auto scales = [&](const uint8_t *row) {  // (rows of scales have 16 bytes less often)
      if constexpr (E == 0) return load16(row + 4 * s, SHIFT >= 1);
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int u = 0; u < 4; u++)
        if (SHIFT == 2 || s + u < end) w[u] = row[min(4 * (s + u) + q, nb - 1)];
      return make_uint4(w[0], w[1], w[2], w[3]);
    };
    uint4 sa[MT], sb[MATS];
#pragma unroll
    for (int t = 0; t < MATS; t++) sb[t] = scales(bs[t]);
#pragma unroll
    for (int i = 0; i < MT; i++) {
      sa[i] = make_uint4(0, 0, 0, 0);
      if (in[i]) sa[i] = scales(as[i]);
    }
    Step x[U];
#pragma unroll
    for (int h = 0; h < 4; h += U) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int k = 64 * (s + h + u) + 16 * q;
        // (a load that is put together here would be waited for here)
        if (E && SHIFT != 2 && s + h + u >= end) break;
#pragma unroll
        for (int t = 0; t < MATS; t++) x[u].b[t] = load(bp[t], k, a.kb);
#pragma unroll
        for (int i = 0; i < MT; i++) {
          x[u].a[i] = make_uint4(0, 0, 0, 0);
          if (in[i]) x[u].a[i] = load(ap[i], k, a.kb);
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (E && s + h + u >= end) break;
        auto byte = [&](const uint4 &v) {
          return (h + u == 0 ? v.x : h + u == 1 ? v.y : h + u == 2 ? v.z : v.w) >> (E ? 0 : 8 * q);
        };
#pragma unroll
        for (int t = 0; t < MATS; t++) x[u].bs[t] = byte(sb[t]);
#pragma unroll
        for (int i = 0; i < MT; i++) x[u].as[i] = byte(sa[i]);
        if (E == 1 && 64 * (s + h + u + 1) > a.kb) {
          const int k = 64 * (s + h + u) + 16 * q;
#pragma unroll
          for (int t = 0; t < MATS; t++) x[u].b[t] = row_shift(x[u].b[t], k, a.kb);
#pragma unroll
          for (int i = 0; i < MT; i++) x[u].a[i] = row_shift(x[u].a[i], k, a.kb);
          // (a block behind the end must not bring the last one's scale, which may be NaN)
#pragma unroll
          for (int t = 0; t < MATS; t++) x[u].bs[t] = k < a.kb ? x[u].bs[t] : 127;
#pragma unroll
          for (int i = 0; i < MT; i++) x[u].as[i] = k < a.kb ? x[u].as[i] : 127;
        }
        run(x[u]);
      }
    }
  };
  int s = wave * span;
  const int end = min(s + span, (a.kb + 63) >> 6);
  for (; 64 * (s + 4) <= a.kb && s < end; s += 4) four(s, end, std::integral_constant<int, 0>{});
  if (s < end) {
    if (a.kb >= 16) four(s, end, std::integral_constant<int, 1>{});
    else four(s, end, std::integral_constant<int, 2>{});
  }
  if (waves > 1) {
#pragma unroll
    for (int t = 0; t < MATS; t++)
#pragma unroll
      for (int i = 0; i < MT; i++) part[(wave * T + t * MT + i) * 64 + lane] = acc[t][i];
    __syncthreads();
  }
  // a wave stores every `waves`-th 16 x 16 tile
  for (int i = wave; i < MT; i += waves) {
    v4f v[MATS];
#pragma unroll
    for (int t = 0; t < MATS; t++) {
      if (waves > 1) {
        v[t] = part[(t * MT + i) * 64 + lane];
        for (int w = 1; w < waves; w++) v[t] += part[(w * T + t * MT + i) * 64 + lane];
      } else {
#pragma unroll
        for (int ii = 0; ii < MT; ii++)
          if (ii == i) v[t] = acc[t][ii];
      }
    }
    const int row = m0 + 16 * i + r, col = n0 + 4 * q;
    if (row >= a.M) continue;
    v4f y = v[0];
    if constexpr (MATS == 2) {
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = swiglu(v[0][e], v[1][e]);
    }
    float *dst = a.out + (int64_t)row * a.ldo + col;
    if (col + 3 < a.N) {
      *(f4any *)dst = y;
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (col + e < a.N) dst[e] = y[e];
    }
  }
}

template <int MT, int MATS>
int launch_skinny(Mx4Args a, hipStream_t st) {
  const int64_t bn = cdiv(a.N, 16), bm = cdiv(a.M, 16 * MT);
  // about twelve waves to a CU, up to 16 to a block (64 KiB of sums)
  const int steps = (a.kb + 63) >> 6;
  int waves = (int)std::min<int64_t>({cdiv(12 * num_cus(), bn * bm), skinny_waves(MT, MATS), std::max(steps, 1), 64 / (MATS * MT)});
  const int span = (int)cdiv(cdiv(steps, waves), 4) * 4;
  if (span) waves = (int)cdiv(steps, span);
  // a launch has below 2^31 threads: in turn, runs of column blocks, and of row blocks where
  // one run has all columns
  const int64_t most = INT32_MAX / (64 * waves), cb = std::min(bn, most), rb = std::max<int64_t>(most / bn, 1);
  KernelTimer kt(st, "mx4_skinny");
  for (int64_t i = 0; i < bm; i += rb) {
    for (int64_t j = 0; j < bn; j += cb) {
      Mx4Args c = a;
      const int64_t row = 16 * MT * i, col = 16 * j;
      const int64_t rows = std::min(16 * MT * rb, a.M - row), cols = std::min(16 * cb, a.N - col);
      c.a += row * a.lda, c.as += row * a.ldas, c.out += row * a.ldo + col, c.M = (int)rows, c.N = (int)cols;
      for (int t = 0; t < MATS; t++) c.b[t] += col * a.ldb[t], c.bs[t] += col * a.ldbs[t];
      const int64_t blocks_n = cdiv(cols, 16);
      hipLaunchKernelGGL((a.shift_codes ? mx4_skinny_k<MT, MATS, 2> : a.shift ? mx4_skinny_k<MT, MATS, 1> : mx4_skinny_k<MT, MATS, 0>),
                         dim3((unsigned)(blocks_n * cdiv(rows, 16 * MT))), dim3(64 * waves),
                         waves > 1 ? waves * MATS * MT * 1024 : 0, st, c, span, (int)blocks_n);
      SIMP_HIP(hipGetLastError());
    }
  }
  return SIMP_RT_OK;
}

// ---- large products: 256 x 256 tiles on an LDS-DMA ring

// dma16 (rt_device.h) from a wave's base address and a lane's offset: one register instead
// of two, so that nothing of the tile kernel's loop is spilled.
__device__ __forceinline__ void dma16_at(const void *base, uint32_t off, uint32_t lds_off) {
  uint32_t saved;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %2, %3\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(saved)
      : "s"(__builtin_amdgcn_readfirstlane(lds_off)), "v"(off), "s"(base)
      : "memory");
}

// The scale bytes of blocks 16g .. 16g + 15 of a row of nb blocks, for four K-steps of 128:
// dword q has block q of the steps 0 .. 3 in its bytes 0 .. 3, so a lane (row, q) keeps
// one register for the four and the matrix instruction picks the step's byte.  Blocks
// behind the row's end get 2^-127: the codes that the last stage reads in their place
// (its first block again) then add up to less than 2^-240, which no sum notices.
__device__ __forceinline__ uint4 scale_group(const uint8_t *s, int g, int nb, bool shift) {
  uint32_t w[4];  // w[j]: blocks 4j .. 4j+3 of the group
  if (16 * g + 16 <= nb) {
    const uint4 v = load16(s + 16 * g, shift);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if (nb >= 4) {  // the row's last four bytes, shifted down
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int b0 = 16 * g + 4 * j, at = min(b0, nb - 4);
      const uint32_t v = *(const u1any *)(s + at);
      w[j] = b0 - at < 4 ? v >> (8 * (b0 - at)) : 0;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = 0;
    for (int e = 0; e < nb && g == 0; e++) w[0] |= (uint32_t)s[e] << (8 * e);
  }
  // 4 x 4 byte transpose
  const uint32_t x0 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u),
                 x1 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u),
                 y0 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u),
                 y1 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
  return make_uint4(__builtin_amdgcn_perm(y0, x0, 0x05040100u),
                    __builtin_amdgcn_perm(y0, x0, 0x07060302u),
                    __builtin_amdgcn_perm(y1, x1, 0x05040100u),
                    __builtin_amdgcn_perm(y1, x1, 0x07060302u));
}

// Scale bytes as the 256 x 256 tiles read them: for 64 rows and a group of four K-steps
// 1 KB, 16 bytes a row (scale_group), so that one DMA instruction brings a wave the scales
// of 64 rows for four steps (8192 + 8192 rows of K = 8192: 4 us).  Row v of W1 and W3 together:
// 16 rows of one, then 16 of the other.
template <int MATS>
__global__ void __launch_bounds__(256)
    mx4_pack_scales_k(const Mx4Args a, uint4 *__restrict__ pa, uint4 *__restrict__ pb, int ga, int groups) {
  const int r = threadIdx.x & 63, g = 4 * blockIdx.y + (threadIdx.x >> 6);
  if (g >= groups) return;
  const bool is_a = (int)blockIdx.x < ga;
  const int rg = is_a ? blockIdx.x : blockIdx.x - ga, v = rg * 64 + r;
  const int mat = !is_a && MATS == 2 ? (v >> 4) & 1 : 0;
  const int row = !is_a && MATS == 2 ? (v >> 5) * 16 + (v & 15) : v;
  const uint8_t *s = is_a ? a.as + (int64_t)row * a.ldas : a.bs[mat] + (int64_t)row * a.ldbs[mat];
  (is_a ? pa : pb)[((int64_t)rg * groups + g) * 64 + r] =
      scale_group(s, g, row < (is_a ? a.M : a.N) ? (a.kb + 15) >> 4 : 0, a.shift);
}

template <int P>
__device__ __forceinline__ v4f mfma_step(const uint4 &b, uint32_t sb, const uint4 &a, uint32_t sa, v4f c) {
  const v8i x = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0},
            y = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(y, x, c, 4, 4, P, (int)sb, P, (int)sa);
}

// Persistent 256 x 256 tiles (MATS == 2: of 128 columns of W1 and W3 each), 8 waves of 128 x
// 64 in K-steps of 64 code bytes.  global_load_lds_dwordx4 fills a ring of two slots of two
// steps each, so that every request is a whole line of 128 bytes: half lines, in four slots
// of one step, cost 8192^3 184 us for the loads alone, not 129 (whole: 267, not 260).
// 8192^3: 254 us, 4.3 POP/s; the matrix instructions take 57% of the cycles at 2.0 GHz, and
// alone, from registers, 164 us, for the clock falls with them (6.7 POP/s).
template <int MATS>
__global__ void __launch_bounds__(512)
    mx4_dma_k(const Mx4Args a, const uint4 *__restrict__ pa, const uint4 *__restrict__ pb,
              int tiles_m, int tiles_n, int groups, int stream, int stagger) {
  constexpr int BM = 256, BN = 256, BK = 128, SLOTS = 2, WGN = 4;  // BK: bytes of a slot's rows
  constexpr int WM = 128, WN = 64, FM = WM / 16, FN = WN / 16;
  constexpr int SLOT = (BM + BN) * BK, SCALES = (BM + BN) * 16;  // bytes
  constexpr int DA = 4, DB = 4, DPW = DA + DB;  // DMA instructions of a wave
  // a group's scales are issued when the group before has been read: one buffer
  __shared__ uint4 lds[(SLOTS * SLOT + SCALES) / 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm0 = (wave / WGN) * WM, wn0 = (wave % WGN) * WN;
  const int nk = (a.kb + 63) / 64, ns = (a.kb + BK - 1) / BK;
  const int ntiles = tiles_m * tiles_n;
  const int lrow = lane & 15, lkc = lane >> 4;
  // chunk c of row r lies at c ^ ((r >> 1) & 7)
  const int drow = lane >> 3, dkc[2] = {16 * ((lane & 7) ^ (lane >> 4)), 16 * ((lane & 7) ^ (4 + (lane >> 4)))};
  const int rslot[2] = {lrow * 8 + (lkc ^ (lrow >> 1)), lrow * 8 + ((4 + lkc) ^ (lrow >> 1))};
  const uint32_t lds0 = lds_offset(lds);
  // Workgroups of equal tiles store at the same time, and all wait for the memory then; with
  // eight starts, `stagger` of about 1 us apart, the others of an XCD compute meanwhile.
  for (int z = stagger * ((blockIdx.x >> 3) & 7); z > 0; z--) __builtin_amdgcn_s_sleep(32);
  const uint32_t *sl = (const uint32_t *)(lds + SLOTS * SLOT / 16) + lrow * 4 + lkc;

  for (int vb = blockIdx.x; vb < ntiles; vb += gridDim.x) {
    int tm, tn;
    tile_of_block(vb, ntiles, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * BM, n0 = tn * (BN / MATS);
    // a lane's rows of the wave's blocks of 8, from the tile's first (B: 16 rows of W1, 16 of W3
    // in turn)
    const uint8_t *baseA = a.a + (int64_t)m0 * a.lda, *baseB[MATS];
#pragma unroll
    for (int t = 0; t < MATS; t++) baseB[t] = a.b[t] + (int64_t)n0 * a.ldb[t];
    uint32_t offA[DA], offB[DB];
#pragma unroll
    for (int i = 0; i < DA; i++)
      offA[i] = (uint32_t)min(8 * (DA * wave + i) + drow, a.M - 1 - m0) * (uint32_t)a.lda + dkc[i & 1];
#pragma unroll
    for (int i = 0; i < DB; i++) {
      const int r = MATS == 2 ? 16 * wave + 8 * (i & 1) + drow : 8 * (DB * wave + i) + drow;
      offB[i] = (uint32_t)min(r, a.N - 1 - n0) * (uint32_t)a.ldb[i / 2 % MATS] + dkc[i & 1];
    }
    // 64 rows of scales to a wave: A's, then B's
    const uint4 *baseS = wave < 4 ? pa + (int64_t)(4 * tm + wave) * groups * 64
                                  : pb + (int64_t)(4 * tn + wave - 4) * groups * 64;
    // Part i of a slot; the scales of a group of four steps go ahead of its first slot.  `last`: s
    // may be the last, which can be shorter.
    auto issue = [&](int s, auto last, int i) {
      const uint32_t st = lds0 + (s & 1) * SLOT;
      const int64_t k0 = (int64_t)s * BK;
      uint32_t back = 0;
      if constexpr (decltype(last)::value) back = k0 + dkc[i & 1] < a.kb ? 0 : dkc[i & 1];
      if (i == 0 && (s & 1) == 0) dma16_at(baseS + (s >> 1) * 64, 16 * lane, lds0 + SLOTS * SLOT + 1024 * wave);
      dma16_at(baseA + k0, offA[i] - back, st + 1024 * (DA * wave + i));
      dma16_at(baseB[i / 2 % MATS] + k0, offB[i] - back, st + BM * BK + 1024 * (DB * wave + i));
    };
    v4f acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
      for (int j = 0; j < FN; j++) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
    uint4 fa[FM], fb[2][FN];
    uint32_t ra[FM], rb[FN], rbn[FN];  // scales of four steps
    // step `at` of the ring's four, 16 rows from 16 blk on (A, then B)
    auto frag = [&](int at, int blk) { return lds[(at >> 1) * (SLOT / 16) + blk * 128 + rslot[at & 1]]; };
    constexpr int BOFF = BM / 16;  // first B block of a slot
    auto scale = [&](int row) { return sl[4 * row]; };
    using T = std::true_type;
    using F = std::false_type;
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));  // the previous tile's stores, and its last reads
    __builtin_amdgcn_s_waitcnt(waitcnt_lgkm0);
    block_barrier();
    for (int p = 0; p < min(SLOTS, ns); p++)
#pragma unroll
      for (int i = 0; i < DA; i++) issue(p, T{}, i);
    if (ns >= SLOTS) __builtin_amdgcn_s_waitcnt(waitcnt_vm(DPW));
    else __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    block_barrier();
#pragma unroll
    for (int j = 0; j < FN; j++) fb[0][j] = frag(0, BOFF + wn0 / 16 + j), rb[j] = scale(BM + wn0 + 16 * j);
#pragma unroll
    for (int i = 0; i < FM; i++) fa[i] = frag(0, wm0 / 16 + i), ra[i] = scale(wm0 + 16 * i);
    // Step kt: the fragments of step kt + 1 are read while the products of step kt run.  In an
    // odd step every wave has read this slot: the next is waited for, and this one filled
    // again, ahead of the products (spread over them 268 us).  Steady: slot kt / 2 + 2 is
    // there and not the last.  (Behind the last step the reads bring stale LDS that is not used.)
    auto step = [&](int kt, auto phase, auto steady) {
      constexpr int P = decltype(phase)::value, cb = P & 1;
      constexpr bool S = decltype(steady)::value;
      if constexpr (P & 1) {
        __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
        __builtin_amdgcn_s_waitcnt(waitcnt_lgkm0);
        block_barrier();
#pragma unroll
        for (int i = 0; i < DA; i++) {
          if constexpr (S) issue((kt >> 1) + 2, F{}, i);
          else if ((kt >> 1) + 2 < ns) issue((kt >> 1) + 2, T{}, i);
        }
      }
      constexpr int next = (P + 1) & 3;
#pragma unroll
      for (int j = 0; j < FN; j++) {
        fb[cb ^ 1][j] = frag(next, BOFF + wn0 / 16 + j);
        if constexpr (P == 3) rbn[j] = scale(BM + wn0 + 16 * j);
      }
#pragma unroll
      for (int i = 0; i < FM; i++) {
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = mfma_step<P>(fb[cb][j], rb[j], fa[i], ra[i], acc[i][j]);
        fa[i] = frag(next, wm0 / 16 + i);
        if constexpr (P == 3) ra[i] = scale(wm0 + 16 * i);
      }
      if constexpr (P == 3) {
#pragma unroll
        for (int j = 0; j < FN; j++) rb[j] = rbn[j];
      }
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I3 = std::integral_constant<int, 3>;
    int kt = 0;
    for (; (kt >> 1) + 4 < ns; kt += 4) {
      step(kt, I0{}, T{});
      step(kt + 1, I1{}, T{});
      step(kt + 2, I2{}, T{});
      step(kt + 3, I3{}, T{});
    }
    for (; kt < nk; kt += 4) {
      step(kt, I0{}, F{});
      if (kt + 1 < nk) step(kt + 1, I1{}, F{});
      if (kt + 2 < nk) step(kt + 2, I2{}, F{});
      if (kt + 3 < nk) step(kt + 3, I3{}, F{});
    }
    // acc[i][j][r] = C[m0 + wm0 + 16 i + l%16][v0 + wn0 + 16 j + 4 (l/16) + r]
    constexpr int NF = FN / MATS;  // fragments side by side in out
    const int col = n0 + (wn0 / MATS) + 16 * (lrow & (NF - 1)) + 4 * lkc;
#pragma unroll
    for (int i = 0; i < FM; i++) {
      v4f v[NF];
#pragma unroll
      for (int j = 0; j < NF; j++) {
        v[j] = acc[i][j * MATS];
        if constexpr (MATS == 2) {
#pragma unroll
          for (int r = 0; r < 4; r++) v[j][r] = swiglu(v[j][r], acc[i][2 * j + 1][r]);
        }
      }
      lane_transpose<NF>(v);
#pragma unroll
      for (int j = 0; j < NF; j++) {
        const int row = m0 + wm0 + 16 * i + (lrow & ~(NF - 1)) + j;
        if (row >= a.M || col >= a.N) continue;
        float *dst = a.out + (int64_t)row * a.ldo + col;
        if (stream) {
          __builtin_nontemporal_store(v[j], (v4f *)dst);
        } else if (col + 3 < a.N) {
          *(f4any *)dst = v[j];
        } else {
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (col + r < a.N) dst[r] = v[j][r];
        }
      }
    }
  }
}

// ---- products between the two: BM x BN tiles, stages of 128 code bytes

// What bounds them is the path that brings the operands into LDS, 16 KB for a 64 x 64 tile and
// stage (200 x 3200 x 8640: 12.2 us a call, 10.9 one behind the other in a graph, 110 MB at about
// 80% of the rate that DMA alone reaches), and below one tile to a CU a stage's round trip.
// (64 bytes of a row to a store instead of 128: 11.5 in a graph; 700 rows 27.4, not 26.0.)
// REG: rows that do not lie on 16 bytes; a stage is loaded as aligned dwords, waits in registers while
// the one before is multiplied, and is put together on its way into LDS.
// KS groups of WGM x WGN waves have a part of K each, with a ring of SLOTS stages of their
// own, and their sums meet in LDS in the order of K: the chain of stages, each of which
// costs a round trip and a barrier, is KS times shorter, and a tile that has a CU to
// itself keeps it busy.  A stage is two K-steps; a DMA instruction is 8 rows of 128 bytes,
// whole lines.  The scales of RG groups of a part are staged through registers into
// LDS as scale_group gives them (RG odd: rows of scales then start in different banks),
// and those of the next RG when they are used up.
template <int BM, int BN, int WGM, int WGN, int KS, int RG, int MATS, bool REG>
__global__ void __launch_bounds__(64 * WGM * WGN * KS)
    mx4_ring_k(const Mx4Args a, int tiles_m, int tiles_n, int per) {
  constexpr int NW = WGM * WGN, NT = 64 * NW * KS;
  constexpr int WM = BM / WGM, WN = BN / WGN, FM = WM / 16, FN = WN / 16;
  constexpr int BK = 128;
  constexpr int SA = BM * BK, SB = BN * BK, STAGE = SA + SB;  // bytes
  constexpr int DA = SA / 1024 / NW, DB = SB / 1024 / NW;     // DMA instructions per wave
  constexpr int SLOTS = 2;
  static_assert(DA >= 1 && DB >= 1 && FN % MATS == 0, "ring shape");
  static_assert(RG % 2 == 1 && BM * BN * 4 <= SLOTS * STAGE, "scales and sums");
  __shared__ uint4 lds[KS * SLOTS * STAGE / 16];
  __shared__ uint4 sc[KS * (BM + BN) * RG];
  const int lane = threadIdx.x & 63, wall = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = wall % NW, part = wall / NW;
  const int wm0 = (wave / WGN) * WM, wn0 = (wave % WGN) * WN;
  const int lrow = lane & 15, lkc = lane >> 4;
  uint4 *ring = lds + part * (SLOTS * STAGE / 16);
  const uint32_t lds_base = lds_offset(ring);
  const int fsw = (lrow >> 1) & 7;  // chunk swizzle of this lane's operand rows
  const int ns = (a.kb + BK - 1) / BK, nb = (a.kb + 15) >> 4;
  const int s0 = part * per, s1 = min(s0 + per, ns);  // this part's stages (per is even)
  int tm, tn;
  tile_of_block(blockIdx.x, tiles_m * tiles_n, tiles_m, tiles_n, tm, tn);
  const int m0 = tm * BM, n0 = tn * (BN / MATS);
  const uint8_t *baseA = a.a + (int64_t)m0 * a.lda;
  const uint8_t *baseB[MATS];
#pragma unroll
  for (int t = 0; t < MATS; t++) baseB[t] = a.b[t] + (int64_t)n0 * a.ldb[t];
  uint32_t offA[DA], offB[DB];
#pragma unroll
  for (int i = 0; i < DA; i++) {
    const int r = 8 * (wave * DA + i) + (lane >> 3);
    offA[i] = (uint32_t)min(r, a.M - 1 - m0) * (uint32_t)a.lda + 16 * ((lane & 7) ^ ((r >> 1) & 7));
  }
#pragma unroll
  for (int i = 0; i < DB; i++) {
    const int v = 8 * (wave * DB + i) + (lane >> 3);
    const int r = MATS == 2 ? (v >> 5) * 16 + (v & 15) : v;
    const int t = MATS == 2 ? ((wave * DB + i) >> 1) & 1 : 0;
    offB[i] = (uint32_t)min(r, a.N - 1 - n0) * (uint32_t)a.ldb[t] + 16 * ((lane & 7) ^ ((v >> 1) & 7));
  }
  // `last`: st may be the last stage, where blocks behind the row's end are its first again
  auto issue = [&](int st, int slot, auto last) {
    const uint32_t dst = lds_base + slot * STAGE;
    const int64_t k0 = (int64_t)st * BK;
    auto go = [&](const uint8_t *base, uint32_t off, int i, uint32_t d) {
      if constexpr (decltype(last)::value) {
        const int c = 16 * ((lane & 7) ^ ((4 * i + (lane >> 4)) & 7));  // the lane's chunk, as above
        off -= k0 + c < a.kb ? 0 : c;
      }
      dma16_at(base + k0, off, d);
    };
#pragma unroll
    for (int i = 0; i < DA; i++) go(baseA, offA[i], wave * DA + i, dst + 1024 * (wave * DA + i));
#pragma unroll
    for (int i = 0; i < DB; i++)
      go(baseB[MATS == 2 ? ((wave * DB + i) >> 1) & 1 : 0], offB[i], wave * DB + i,
         dst + SA + 1024 * (wave * DB + i));
  };
  // REG: a stage's pieces on their way through registers, as aligned dwords, and into the slot.
  struct Piece {
    uint4 u;
    uint32_t w, sh;
  };
  Piece pieces[REG ? DA + DB : 1];
  // the bytes of a lane's piece i that lie behind the row's end
  auto behind = [&](int st, int i) {
    return max(st * BK + 16 * ((lane & 7) ^ ((4 * i + (lane >> 4)) & 7)) + 16 - a.kb, 0);
  };
  auto fetch = [&](int st, auto last) {
    const int64_t k0 = (int64_t)st * BK;
    auto go = [&](const uint8_t *base, uint32_t off, int i, Piece &x) {
      const uint8_t *p = base + k0 + off;
      if constexpr (decltype(last)::value) p -= behind(st, i);
      x.sh = (uintptr_t)p & 3;
      const u4any u = *(const u4any *)__builtin_assume_aligned(p - x.sh, 4);
      x.u = make_uint4(u.x, u.y, u.z, u.w), x.w = *(const u1any *)(p + 12);
    };
#pragma unroll
    for (int i = 0; i < DA; i++) go(baseA, offA[i], wave * DA + i, pieces[i]);
#pragma unroll
    for (int i = 0; i < DB; i++)
      go(baseB[MATS == 2 ? ((wave * DB + i) >> 1) & 1 : 0], offB[i], wave * DB + i, pieces[DA + i]);
  };
  auto put = [&](int st, int slot, auto last) {
#pragma unroll
    for (int i = 0; i < DA + DB; i++) {
      const Piece &x = pieces[i];
      const int at = i < DA ? wave * DA + i : wave * DB + i - DA;
      uint4 v = make_uint4(__builtin_amdgcn_alignbyte(x.u.y, x.u.x, x.sh), __builtin_amdgcn_alignbyte(x.u.z, x.u.y, x.sh),
                           __builtin_amdgcn_alignbyte(x.u.w, x.u.z, x.sh), x.w);
      if constexpr (decltype(last)::value) v = shift_down(v, min(behind(st, at), 16));
      ring[slot * (STAGE / 16) + (i < DA ? 0 : SA / 16) + at * 64 + lane] = v;
    }
  };
  // (slot and row part constant: the reads' immediate offsets)
  const uint4 *fA[2], *fB[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    fA[h] = ring + wm0 * 8 + lrow * 8 + ((4 * h + lkc) ^ fsw);
    fB[h] = fA[h] + (BM + wn0 - wm0) * 8;
  }
  const uint32_t *sl = (const uint32_t *)(sc + part * (BM + BN) * RG) + lrow * 4 * RG + lkc;
  auto scale = [&](int g, int row) { return sl[row * 4 * RG + 4 * g]; };
  v4f acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; i++)
#pragma unroll
    for (int j = 0; j < FN; j++) acc[i][j] = v4f{0.f, 0.f, 0.f, 0.f};
  using T = std::true_type;
  using F = std::false_type;
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;

  // the row whose scales this thread stages: A's, then B's, of every part
  constexpr int ROWS = KS * (BM + BN), TPR = NT / ROWS > 0 ? NT / ROWS : 1, U = (RG + TPR - 1) / TPR;
  static_assert(NT >= ROWS, "a thread to each row");
  const int srow = threadIdx.x % ROWS, sg = threadIdx.x / ROWS;
  const uint8_t *sp;
  {
    const int p = srow / (BM + BN), row = srow - p * (BM + BN);
    if (row < BM) {
      sp = a.as + (int64_t)min(m0 + row, a.M - 1) * a.ldas;
    } else {
      const int v = row - BM, r = MATS == 2 ? (v >> 5) * 16 + (v & 15) : v;
      const int64_t n = min(n0 + r, a.N - 1);
      sp = MATS == 2 && (v & 16) ? a.bs[MATS - 1] + n * a.ldbs[MATS - 1] : a.bs[0] + n * a.ldbs[0];
    }
    sp += 8 * p * per;  // a stage is 8 blocks
  }
  const int snb = nb - 8 * (srow / (BM + BN)) * per;  // the row's blocks from there on

  for (int d0 = 0; d0 < per; d0 += 2 * RG) {  // spans of every part whose scales are staged
    const int len = min(per - d0, 2 * RG), groups = len >> 1;  // the same for all parts
    const int c0 = s0 + d0, c1 = min(c0 + len, s1);
    if (d0) block_barrier();  // the span before is read
    const int first = max(min(SLOTS, c1 - c0), 0);
    if constexpr (REG) {
      if (first > 0) fetch(c0, T{}), put(c0, 0, T{});
      if (first > 1) fetch(c0 + 1, T{});
    } else {
      for (int i = 0; i < first; i++) issue(c0 + i, i, T{});
    }
    // scales: a thread has one row (and part) and takes its groups all at once
    uint4 sv[U];
#pragma unroll
    for (int u = 0; u < U; u++)
      if (u * TPR + sg < groups) sv[u] = scale_group(sp, (d0 >> 1) + u * TPR + sg, snb, a.shift);
#pragma unroll
    for (int u = 0; u < U; u++)
      if (u * TPR + sg < groups) sc[srow * RG + u * TPR + sg] = sv[u];
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
    lds_barrier();
    uint4 fra[2][FM], frb[2][FN];
    uint32_t sa[FM], sb[FN], na[FM], nb_[FN];
    auto read = [&](auto slot, auto half) {
      constexpr int h = decltype(half)::value, at = decltype(slot)::value * (STAGE / 16);
#pragma unroll
      for (int j = 0; j < FN; j++) frb[h][j] = fB[h][at + j * 128];
#pragma unroll
      for (int i = 0; i < FM; i++) fra[h][i] = fA[h][at + i * 128];
    };
    auto mul = [&](auto phase) {
      constexpr int P = decltype(phase)::value, h = P & 1;
#pragma unroll
      for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = mfma_step<P>(frb[h][j], sb[j], fra[h][i], sa[i], acc[i][j]);
    };
#pragma unroll
    for (int j = 0; j < FN; j++) sb[j] = scale(0, BM + wn0 + 16 * j);
#pragma unroll
    for (int i = 0; i < FM; i++) sa[i] = scale(0, wm0 + 16 * i);
    read(I0{}, I0{});
    // Stage st: its second step is read while its first is multiplied; then stage st + 1
    // is waited for, stage st is read on every wave, and its slot is filled again while
    // the second step is multiplied.  (c0 is even: an even stage lies in slot 0.)
    // Steady: stage st + 2 is there and not the last.  (Reads behind the last stage and
    // group bring stale LDS that is not used.)  One barrier a stage, in every part.  The
    // scheduling barriers keep the reads ahead of the products that they run beside.
    auto stage = [&](int st, auto odd, auto steady) {
      constexpr int o = decltype(odd)::value;
      constexpr bool S = decltype(steady)::value;
      using Other = std::integral_constant<int, o ^ 1>;
      const bool in = S || st < c1;  // (a part may have fewer stages)
      read(odd, I1{});
      __builtin_amdgcn_sched_barrier(0);
      if (in) mul(std::integral_constant<int, 2 * o>{});
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (REG) {
        if constexpr (S) put(st + 1, o ^ 1, F{});
        else if (st + 1 < c1) put(st + 1, o ^ 1, T{});
        lds_barrier();
      } else {
        __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
        __builtin_amdgcn_s_waitcnt(waitcnt_lgkm0);
        block_barrier();
      }
      read(Other{}, I0{});
      if constexpr (o == 1) {
        const int g = min((st + 1 - c0) >> 1, RG - 1);
#pragma unroll
        for (int j = 0; j < FN; j++) nb_[j] = scale(g, BM + wn0 + 16 * j);
#pragma unroll
        for (int i = 0; i < FM; i++) na[i] = scale(g, wm0 + 16 * i);
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (REG) {
        if constexpr (S) fetch(st + 2, F{});
        else if (st + 2 < c1) fetch(st + 2, T{});
      } else {
        if constexpr (S) issue(st + 2, o, F{});
        else if (st + 2 < c1) issue(st + 2, o, T{});
      }
      if (in) mul(std::integral_constant<int, 2 * o + 1>{});
      if constexpr (o == 1) {
#pragma unroll
        for (int j = 0; j < FN; j++) sb[j] = nb_[j];
#pragma unroll
        for (int i = 0; i < FM; i++) sa[i] = na[i];
      }
    };
    int st = c0;
    for (; st + 4 < c1; st += 2) {
      stage(st, I0{}, T{});
      stage(st + 1, I1{}, T{});
    }
    for (; st < c0 + len; st += 2) {
      stage(st, I0{}, F{});
      stage(st + 1, I1{}, F{});
    }
  }
  // acc[i][j][r] = C[m0 + wm0 + 16 i + l%16][v0 + wn0 + 16 j + 4 (l/16) + r]; the parts share the
  // wave's fragments out between them, NF side by side in out
  constexpr int NF = FN / MATS;
  v4f *sums = (v4f *)lds;  // [part][wave][i][j][lane]
  if constexpr (KS > 1) {
    lds_barrier();  // every wave is through with its ring
#pragma unroll
    for (int i = 0; i < FM; i++)
#pragma unroll
      for (int j = 0; j < FN; j++) sums[((part * NW + wave) * FM * FN + i * FN + j) * 64 + lane] = acc[i][j];
    lds_barrier();
  }
  auto sum = [&](int i, int j) {
    if constexpr (KS == 1) return acc[i][j];
    v4f v = sums[(wave * FM * FN + i * FN + j) * 64 + lane];
#pragma unroll
    for (int p = 1; p < KS; p++) v += sums[((p * NW + wave) * FM * FN + i * FN + j) * 64 + lane];
    return v;
  };
#pragma unroll
  for (int o = 0; o < FM; o += KS) {
    if (KS > 1 && o + part >= FM) break;
    const int i = KS > 1 ? o + part : o;
    v4f v[NF];
#pragma unroll
    for (int j = 0; j < NF; j++) {
      v[j] = sum(i, j * MATS);
      if constexpr (MATS == 2) {
        const v4f w = sum(i, j * MATS + 1);
#pragma unroll
        for (int r = 0; r < 4; r++) v[j][r] = swiglu(v[j][r], w[r]);
      }
    }
    if constexpr (NF > 1) lane_transpose<NF>(v);
    const int col = n0 + wn0 / MATS + 16 * (lrow & (NF - 1)) + 4 * lkc;
#pragma unroll
    for (int j = 0; j < NF; j++) {
      const int row = m0 + wm0 + 16 * i + (lrow & ~(NF - 1)) + j;
      if (row >= a.M || col >= a.N) continue;
      float *dst = a.out + (int64_t)row * a.ldo + col;
      if (col + 3 < a.N) {
        *(f4any *)dst = v[j];
      } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
          if (col + r < a.N) dst[r] = v[j][r];
      }
    }
  }
}

template <int BM, int BN, int WGM, int WGN, int KS, int RG, int MATS, bool REG>
int launch_ring(const Mx4Args &a, hipStream_t st) {
  const int64_t tm = cdiv(a.M, BM), tn = cdiv(a.N, BN / MATS);
  const int per = (int)(2 * cdiv(cdiv(a.kb, 128), 2 * KS));  // stages of a part, even
  static const char *const kNames[2][3] = {{"mx4_ring64", "mx4_ring64x2", "mx4_ring128"},
                                           {"mx4_ring64d", "mx4_ring64x2d", "mx4_ring128d"}};
  KernelTimer kt(st, kNames[REG][BN == 128 ? 2 : KS - 1]);
  hipLaunchKernelGGL((mx4_ring_k<BM, BN, WGM, WGN, KS, RG, MATS, REG>), dim3((unsigned)(tm * tn)),
                     dim3(64 * WGM * WGN * KS), 0, st, a, (int)tm, (int)tn, per);
  SIMP_HIP(hipGetLastError());
  return SIMP_RT_OK;
}

// Codes of rows whose bytes the tile kernels cannot read in place (any address and length)
// into rows of whole aligned 16 bytes, zeros behind their ends: A's, then each B's (717 and 2051
// rows of 767 bytes: 4 us).
template <int MATS>
__global__ void __launch_bounds__(256) mx4_pad_k(const Mx4Args a, uint4 *__restrict__ out, int per, int ga, int gb) {
  const int w = (int)blockIdx.x < ga ? 0 : MATS == 2 && (int)blockIdx.x >= ga + gb ? 2 : 1;
  const int64_t first = (int64_t)((int)blockIdx.x - (w > 0 ? ga : 0) - (w > 1 ? gb : 0)) * 256;
  const int64_t ca = (int64_t)a.M * per, cb = (int64_t)a.N * per;
  if (first + threadIdx.x >= (w ? cb : ca)) return;
  int64_t row, c;
  BlockAt(first, per).get(threadIdx.x, row, c);
  const uint8_t *p = w == 0 ? a.a + row * a.lda
                            : a.b[w > 1 ? MATS - 1 : 0] + row * a.ldb[w > 1 ? MATS - 1 : 0];
  out[(w > 0 ? ca : 0) + (w > 1 ? cb : 0) + first + threadIdx.x] = row_shift(row_load(p, 16 * (int)c, a.kb), 16 * (int)c, a.kb);
}

// 256 x 256 tiles; false where their scales cannot be packed (no memory, or a captured call
// whose warm-up left too little).
template <int MATS>
bool launch_dma(const Mx4Args &a, hipStream_t st, int *rc) {
  const int64_t tm = cdiv(a.M, 256), tn = cdiv(a.N, 256 / MATS);
  const int groups = (int)cdiv(a.kb, 256), ga = (int)(4 * tm), gb = (int)(4 * tn);
  const int64_t rgs = (int64_t)(ga + gb) * groups;
  Workspace ws;
  void *p;
  if (tm * tn > INT32_MAX || (int64_t)(ga + gb) * 256 > INT32_MAX || groups > 4 * 65535 ||
      !ws.try_get(st, (size_t)rgs * 1024, &p, 10))
    return false;
  uint4 *pa = (uint4 *)p, *pb = pa + (int64_t)ga * groups * 64;
  hipLaunchKernelGGL(mx4_pack_scales_k<MATS>, dim3((unsigned)(ga + gb), (unsigned)cdiv(groups, 4)),
                     dim3(256), 0, st, a, pa, pb, ga, groups);
  // past the caches only where lines are whole (6276 x 384 x 26422 gated, rows on 8 bytes: 248 us, 363
  // past them; x 26432: 188, 226 into them)
  const int stream = a.N % 16 == 0 && ((uintptr_t)a.out & 63) == 0 && a.ldo % 16 == 0;
  const int64_t grid = std::min<int64_t>(tm * tn, num_cus());
  // (in a graph, without: 8192^3 270 us, 286; 8192 x 256 x 8192 61, 84; 6000 x 1024 x 6000 53, 55;
  // gated 4096 x 2048 x 8192 89, 103; 8192 x 768 x 8192 110, 120; 8192 x 256 x 8192 69, 85)
  const int stagger = tm * tn >= 2 * grid && MATS == 1 ? 2 : tm * tn >= 4 * grid ? 1 : 0;
  KernelTimer kt(st, "mx4_dma");
  hipLaunchKernelGGL((mx4_dma_k<MATS>), dim3((unsigned)grid), dim3(512), 0, st, a, pa, pb, (int)tm,
                     (int)tn, groups, stream, stagger);
  const hipError_t e = hipGetLastError();
  *rc = e == hipSuccess ? SIMP_RT_OK : hip_fail(e, "launch");
  return true;
}

// What each form takes in us, fitted to whole calls (graph replay) of 1 to 8192 rows,
// K = 768 to 8192 and up to 32000 columns; `steps` of 128 elements.
// Over 168 products and gates of 1 to 8192 rows the chosen form takes 1% longer than the best one at
// the median and 9% at the ninetieth percentile; the most are 32% (gated, 300 x 768 x 2048: 7.0 us,
// 64 x 64 tiles 5.3; 64 x 8192 x 8192: 21.7, K in two parts 16.5).
enum Form { kSkinny, kRing64, kRing64x2, kRing128, kTiles256 };
// What the tile kernels make of rows that do not lie on 16 bytes: they read them as dwords
// (the rings' stages go through registers, and take about twice as long: 60 x 2899 x 23360
// gated 23 us, with the copy 40, on 16 bytes 16), or rows are copied first (600 x 3201 x 8640 39.5
// us; as dwords 41).
enum Rows { kDirect, kDwords, kPadded };
struct Choice {
  Form form;
  Rows rows;
};
// `can`: kDirect where rows do lie on 16 bytes, kPadded where they cannot be read as dwords.  Then
// the choice is the one of rows in place: the copy comes on top of every form but the few-row one,
// whose loads take longer in turn (first byte off 4 bytes, 16 x 8640 x 32000: 77 us with the
// copy, 95 without; 64 x 3200 x 8640 gated 24 and 31; 64 x 3200 x 2800 13 and 11, the wrong one).
template <int MATS>
Choice pick(const Mx4Args &a, int64_t cus, Rows can) {
  const double steps = (double)cdiv(a.kb, 64), out = 4e-6 * a.M * a.N / 6.5;
  const int mt = a.M <= 16 ? 16 : a.M <= 32 ? 32 : 64;
  auto tiles = [&](int m, int n) { return cdiv(a.M, m) * cdiv(a.N, n / MATS); };
  auto rounds = [&](int64_t t) { return (double)cdiv(t, cus); };
  const double mem = (a.M + (double)MATS * a.N) * steps * 68 / 5.2e6;  // the operands' time from memory
  // a block's operands from the caches, 33 KB a us to a CU: every row block reads B, every
  // column block A
  const double blocks = (double)cdiv(a.M, mt) * cdiv(a.N, 16) / cus;
  const double cache = std::max(1., blocks) * (std::min(a.M, mt) + 16 * MATS) * steps * 68 / 33.2e3;
  const int64_t t64 = tiles(64, 64), t128 = tiles(64, 128), t256 = tiles(256, 256);
  // outputs' time to memory, and the ends of tiles that nothing hides
  const double out64 = out + (MATS == 2 ? 0.45 : 0.2) * rounds(t64), out128 = out + (MATS == 2 ? 0.55 : 0.1) * rounds(t128);
  const double out256 = out + (MATS == 2 ? 2. * (rounds(t256) - 1) - 1. : 0.);
  double us[5] = {2.5 + std::max(cache, mem) + out,
                  3.5 + std::max(mem, steps / 2 * std::max(0.33, 0.23 * rounds(t64))) + out64,
                  3.8 + std::max(mem, steps / 2 * 0.2 * (t64 <= cus ? 1. : 1.3 * rounds(t64))) + out64,
                  4.0 + std::max(mem, steps / 2 * 0.42 * rounds(t128)) + out128,
                  8.0 + steps * (0.95 * (t256 / cus) + (t256 % cus ? 0.6 + 0.35 * (t256 % cus) / cus : 0.)) + out256};
  const auto least = [](const double *v) { return (int)(std::min_element(v, v + 5) - v); };
  if (can != kDwords) return {(Form)least(us), can};
  const double copy = 6 + (a.M + (double)MATS * a.N) * 2 * a.kb / 4.5e6;
  us[kSkinny] = 2.5 + std::max((a.shift_codes ? 1.9 : a.M > 32 ? 1.6 : 1.1) * cache, (a.shift_codes ? 1.45 : 1.) * mem) + out;
  for (int f = kRing64; f <= kTiles256; f++) us[f] += copy;
  const double dwords[5] = {us[kSkinny],
                            3.5 + std::max(mem, steps / 2 * std::max(0.6, 0.45 * rounds(t64))) + out64,
                            3.8 + std::max(mem, steps / 2 * 0.5 * (t64 <= cus ? 1. : 1.6 * rounds(t64))) + out64,
                            4.0 + std::max(mem, steps / 2 * (t128 <= cus ? 0.82 : 0.95 * rounds(t128))) + out128,
                            us[kTiles256]};
  const int f = least(us), d = least(dwords);
  return us[f] <= dwords[d] ? Choice{(Form)f, kPadded} : Choice{(Form)d, kDwords};
}

// A form on tiles; false where its grid has no room.
template <int MATS, bool REG>
bool launch_tiles(const Mx4Args &a, Form f, hipStream_t st, int *rc) {
  if (!REG && f == kTiles256 && launch_dma<MATS>(a, st, rc)) return true;
  if (cdiv(a.M, 64) * cdiv(a.N, 64 / MATS) > INT32_MAX / 512) return false;
  *rc = f == kRing64 ? launch_ring<64, 64, 2, 2, 1, 9, MATS, REG>(a, st)
        : f == kRing64x2 ? launch_ring<64, 64, 2, 2, 2, 9, MATS, REG>(a, st)
                         : launch_ring<64, 128, 2, 4, 1, 9, MATS, REG>(a, st);
  return true;
}

template <int MATS>
int launch_mx4(const Mx4Args &a, hipStream_t st) {
  int rc;
  // the tile kernels' offsets within a tile are 32-bit
  uintptr_t base = (uintptr_t)a.a, rows = (uintptr_t)a.lda | (uintptr_t)a.kb;
  for (int t = 0; t < MATS; t++) base |= (uintptr_t)a.b[t], rows |= (uintptr_t)a.ldb[t];
  const bool near = std::max({a.lda, a.ldb[0], a.ldb[MATS - 1]}) < (1 << 23);
  const Rows can = near && ((base | rows) & 15) == 0 ? kDirect
                   : near && (base & 3) == 0 && a.kb >= 16 ? kDwords : kPadded;
  const Choice c = pick<MATS>(a, num_cus(), can);
  if (c.form != kSkinny && a.kb > 0) {
    if (c.rows == kDirect) {
      if (launch_tiles<MATS, false>(a, c.form, st, &rc)) return rc;
    } else if (c.rows == kDwords) {
      if (launch_tiles<MATS, true>(a, c.form, st, &rc)) return rc;
    } else if (a.kb < (1 << 23) - 16) {
      const int per = (int)cdiv(a.kb, 16);
      const int64_t ca = (int64_t)a.M * per, cb = (int64_t)a.N * per;
      Workspace ws;
      void *p;
      const int64_t ga = cdiv(ca, 256), gb = cdiv(cb, 256);
      // (no more than 4 GiB, which stay the library's)
      if ((ga + MATS * gb) * 256 <= INT32_MAX && ca + MATS * cb <= (1 << 28) &&
          ws.try_get(st, 16 * (size_t)(ca + MATS * cb), &p, 11)) {
        uint4 *q = (uint4 *)p;
        hipLaunchKernelGGL(mx4_pad_k<MATS>, dim3((unsigned)(ga + MATS * gb)), dim3(256), 0, st, a, q, per,
                           (int)ga, (int)gb);
        SIMP_HIP(hipGetLastError());
        Mx4Args o = a;
        o.a = (const uint8_t *)q, o.lda = 16 * (int64_t)per;
        for (int t = 0; t < MATS; t++)
          o.b[t] = (const uint8_t *)(q + ca + t * cb), o.ldb[t] = 16 * (int64_t)per;
        if (launch_tiles<MATS, false>(o, c.form, st, &rc)) return rc;
      }
      if (can == kDwords && launch_tiles<MATS, true>(a, c.form, st, &rc)) return rc;  // no room for copies
    }
  }
  if (a.M <= 16) return launch_skinny<1, MATS>(a, st);
  if (a.M <= 32) return launch_skinny<2, MATS>(a, st);
  return launch_skinny<4, MATS>(a, st);
}

// ------------------------------------------------------------- entry points

// A rank-2 descriptor and its extent.  One row may have any stride.
template <class T>
struct Mat {
  T *p;
  int64_t off, s[2], st[2], span;
  int check(const char *name) {
    if (s[0] == 1) st[0] = s[1];
    if (s[1] == 1) st[1] = 1;
    if (const int rc = check_descn(name, p, off, 2, s, st, &span)) return rc;
    if (s[0] > INT32_MAX - 4096 || s[1] > INT32_MAX - 4096)
      return set_error(SIMP_RT_EUNSUPPORTED, "%s: dimension above 2^31 - 4097", name);
    return SIMP_RT_OK;
  }
  T *data() const { return p + off; }
  size_t bytes() const { return (size_t)span * sizeof(T); }
  // (an array's rows may lie between those of another output, of this call or of another thread's)
  void rows_of(Operand &o) const { o.set_rows(1, 0, s[0], st[0] * (int64_t)sizeof(T), (size_t)s[1] * sizeof(T)); }
};

// Whether two arrays share an element: ranges that meet do not where both have rows of
// one stride in bytes and each row lies in the gap between the other's.
template <class T, class U>
bool meets(const Mat<T> &a, const Mat<U> &b) {
  if (!overlap(a.data(), a.bytes(), b.data(), b.bytes())) return false;
  const int64_t st = a.st[0] * (int64_t)sizeof(T);
  if (a.s[0] <= 1 || b.s[0] <= 1 || st != b.st[0] * (int64_t)sizeof(U)) return true;
  const uintptr_t x = (uintptr_t)a.data(), y = (uintptr_t)b.data();
  const int64_t d = y >= x ? (int64_t)((y - x) % (uintptr_t)st)
                           : (st - (int64_t)((x - y) % (uintptr_t)st)) % st;
  return d < a.s[1] * (int64_t)sizeof(T) || d + b.s[1] * (int64_t)sizeof(U) > st;
}

// K of the codes' bytes and the scales that go with them.
int check_rows(const char *fn, const char *name, const Mat<const uint8_t> &c,
               const Mat<const uint8_t> &s) {
  if (s.s[0] != c.s[0] || s.s[1] != cdiv(c.s[1], 16))
    return set_error(SIMP_RT_EINVAL,
                     "%s: %s: shape mismatch, codes [%lld,%lld] and scales [%lld,%lld] (one for 16 bytes)",
                     fn, name, (long long)c.s[0], (long long)c.s[1], (long long)s.s[0], (long long)s.s[1]);
  return SIMP_RT_OK;
}

template <int MATS>
int product(const char *fn, Mat<const uint8_t> &a, Mat<const uint8_t> &as,
            Mat<const uint8_t> (&b)[MATS], Mat<const uint8_t> (&bs)[MATS], Mat<float> &o) {
  static const char *const kB[2][2] = {{"b", "w1"}, {"", "w3"}},
                           *const kS[2][2] = {{"b_scales", "s1"}, {"", "s3"}};
  int rc;
  if ((rc = a.check("a")) || (rc = as.check("a_scales")) || (rc = o.check("out")) ||
      (rc = check_rows(fn, "a", a, as)))
    return rc;
  for (int t = 0; t < MATS; t++) {
    const char *name = kB[t][MATS - 1];
    if ((rc = b[t].check(name)) || (rc = bs[t].check(kS[t][MATS - 1])) ||
        (rc = check_rows(fn, name, b[t], bs[t])))
      return rc;
    if (b[t].s[1] != a.s[1] || b[t].s[0] != o.s[1] || a.s[0] != o.s[0])
      return set_error(SIMP_RT_EINVAL, "%s: shape mismatch a[%lld,%lld] %s[%lld,%lld] out[%lld,%lld]",
                       fn, (long long)a.s[0], (long long)a.s[1], name, (long long)b[t].s[0],
                       (long long)b[t].s[1], (long long)o.s[0], (long long)o.s[1]);
  }
  if (o.s[0] == 0 || o.s[1] == 0) return SIMP_RT_OK;
  bool shared = meets(o, a) || meets(o, as);
  for (int t = 0; t < MATS; t++) shared = shared || meets(o, b[t]) || meets(o, bs[t]);
  if (shared) return set_error(SIMP_RT_EINVAL, "%s: out shares memory with another operand", fn);
  const int dev = ensure_device();
  if (dev < 0) return dev;
  Operand oa, oas, ob[MATS], obs[MATS], oo;
  if ((rc = bind_here(oa, a.data(), a.bytes(), Operand::kIn, dev, "a")) ||
      (rc = bind_here(oas, as.data(), as.bytes(), Operand::kIn, dev, "a_scales")) ||
      (rc = bind_here(oo, o.data(), o.bytes(), Operand::kOut, dev, "out")))
    return rc;
  o.rows_of(oo);
  Mx4Args g{};
  g.a = (const uint8_t *)oa.dev(), g.as = (const uint8_t *)oas.dev();
  g.lda = a.st[0], g.ldas = as.st[0];
  for (int t = 0; t < MATS; t++) {
    if ((rc = bind_here(ob[t], b[t].data(), b[t].bytes(), Operand::kIn, dev, kB[t][MATS - 1])) ||
        (rc = bind_here(obs[t], bs[t].data(), bs[t].bytes(), Operand::kIn, dev, kS[t][MATS - 1])))
      return rc;
    g.b[t] = (const uint8_t *)ob[t].dev(), g.bs[t] = (const uint8_t *)obs[t].dev();
    g.ldb[t] = b[t].st[0], g.ldbs[t] = bs[t].st[0];
  }
  g.out = (float *)oo.dev(), g.ldo = o.st[0];
  g.M = (int)o.s[0], g.N = (int)o.s[1], g.kb = (int)a.s[1];
  uintptr_t base = (uintptr_t)g.as, rows = (uintptr_t)g.ldas, cbase = (uintptr_t)g.a, crows = (uintptr_t)g.lda;
  for (int t = 0; t < MATS; t++) {
    base |= (uintptr_t)g.bs[t], rows |= (uintptr_t)g.ldbs[t];
    cbase |= (uintptr_t)g.b[t], crows |= (uintptr_t)g.ldb[t];
  }
  g.shift = (base & 3) == 0 && (rows & 3) != 0;
  g.shift_codes = ((base | cbase) & 3) == 0 && (crows & 3) != 0;
  if ((rc = launch_mx4<MATS>(g, cur_stream()))) return rc;
  Operand *ops[] = {&oa, &oas, &oo, &ob[0], &obs[0], &ob[MATS - 1], &obs[MATS - 1]};
  return finish(ops, 3 + 2 * MATS);
}

// Launches a kernel over the blocks of rows.
struct BlockLaunch {
  int64_t blocks;
  int run;
  unsigned grid;
  int plan(const char *fn, int64_t rows, int64_t per_row) {
    blocks = rows * per_row;
    run = blocks <= (1 << 15) ? 1 : 4;
    const int64_t g = cdiv(blocks, 32 * run);
    if (g > INT32_MAX / 256) return set_error(SIMP_RT_EUNSUPPORTED, "%s: more elements than the grid holds", fn);
    grid = (unsigned)g;
    return SIMP_RT_OK;
  }
};

// Values that go past the caches: too many to stay there for the next operator, rows on 16 bytes.
bool streams(const void *p, int64_t ld, int64_t n) {
  return n >= (int64_t(1) << 24) && ((uintptr_t)p & 15) == 0 && (ld & 3) == 0;
}

}  // namespace
}  // namespace simp

using namespace simp;

extern "C" {

int32_t simp_rt_quantize_mx4(
    const float *x_alloc, const float *x, int64_t x_off, int64_t x_s0, int64_t x_s1, int64_t x_st0,
    int64_t x_st1, uint8_t *c_alloc, uint8_t *codes, int64_t c_off, int64_t c_s0, int64_t c_s1,
    int64_t c_st0, int64_t c_st1, uint8_t *s_alloc, uint8_t *scales, int64_t s_off, int64_t s_s0,
    int64_t s_s1, int64_t s_st0, int64_t s_st1) {
  (void)x_alloc; (void)c_alloc; (void)s_alloc;
  static const char *fn = "quantize_mx4";
  Mat<const float> mx{x, x_off, {x_s0, x_s1}, {x_st0, x_st1}, 0};
  Mat<uint8_t> mc{codes, c_off, {c_s0, c_s1}, {c_st0, c_st1}, 0};
  Mat<uint8_t> ms{scales, s_off, {s_s0, s_s1}, {s_st0, s_st1}, 0};
  int rc;
  if ((rc = mx.check("x")) || (rc = mc.check("codes")) || (rc = ms.check("scales"))) return rc;
  if (c_s0 != x_s0 || s_s0 != x_s0 || c_s1 != cdiv(x_s1, 2) || s_s1 != cdiv(x_s1, 32))
    return set_error(SIMP_RT_EINVAL,
                     "%s: shape mismatch x[%lld,%lld] codes[%lld,%lld] scales[%lld,%lld]", fn,
                     (long long)x_s0, (long long)x_s1, (long long)c_s0, (long long)c_s1,
                     (long long)s_s0, (long long)s_s1);
  if (x_s0 == 0 || x_s1 == 0) return SIMP_RT_OK;
  if (meets(mc, mx) || meets(ms, mx) || meets(mc, ms))
    return set_error(SIMP_RT_EINVAL, "%s: codes or scales share memory with another operand", fn);
  BlockLaunch bl;
  if ((rc = bl.plan(fn, x_s0, s_s1))) return rc;
  const int dev = ensure_device();
  if (dev < 0) return dev;
  Operand ox, oc, os;
  if ((rc = bind_here(ox, mx.data(), mx.bytes(), Operand::kIn, dev, "x")) ||
      (rc = bind_here(oc, mc.data(), mc.bytes(), Operand::kOut, dev, "codes")) ||
      (rc = bind_here(os, ms.data(), ms.bytes(), Operand::kOut, dev, "scales")))
    return rc;
  mc.rows_of(oc), ms.rows_of(os);
  auto kernel = bl.run == 1 ? quantize_mx4_k<1, false>
                : streams(ox.dev(), mx.st[0], x_s0 * x_s1) ? quantize_mx4_k<4, true> : quantize_mx4_k<4, false>;
  hipLaunchKernelGGL(kernel, dim3(bl.grid), dim3(256), 0, cur_stream(), (const float *)ox.dev(), mx.st[0],
                     (uint8_t *)oc.dev(), mc.st[0], (uint8_t *)os.dev(), ms.st[0], x_s1, s_s1, bl.blocks);
  SIMP_HIP(hipGetLastError());
  Operand *ops[] = {&ox, &oc, &os};
  return finish(ops, 3);
}

int32_t simp_rt_dequantize_mx4(
    const uint8_t *c_alloc, const uint8_t *codes, int64_t c_off, int64_t c_s0, int64_t c_s1,
    int64_t c_st0, int64_t c_st1, const uint8_t *s_alloc, const uint8_t *scales, int64_t s_off,
    int64_t s_s0, int64_t s_s1, int64_t s_st0, int64_t s_st1, float *out_alloc, float *out,
    int64_t out_off, int64_t out_s0, int64_t out_s1, int64_t out_st0, int64_t out_st1) {
  (void)c_alloc; (void)s_alloc; (void)out_alloc;
  static const char *fn = "dequantize_mx4";
  Mat<const uint8_t> mc{codes, c_off, {c_s0, c_s1}, {c_st0, c_st1}, 0};
  Mat<const uint8_t> ms{scales, s_off, {s_s0, s_s1}, {s_st0, s_st1}, 0};
  Mat<float> mo{out, out_off, {out_s0, out_s1}, {out_st0, out_st1}, 0};
  int rc;
  if ((rc = mc.check("codes")) || (rc = ms.check("scales")) || (rc = mo.check("out"))) return rc;
  if (c_s0 != out_s0 || s_s0 != out_s0 || c_s1 != cdiv(out_s1, 2) || s_s1 != cdiv(out_s1, 32))
    return set_error(SIMP_RT_EINVAL,
                     "%s: shape mismatch codes[%lld,%lld] scales[%lld,%lld] out[%lld,%lld]", fn,
                     (long long)c_s0, (long long)c_s1, (long long)s_s0, (long long)s_s1,
                     (long long)out_s0, (long long)out_s1);
  if (out_s0 == 0 || out_s1 == 0) return SIMP_RT_OK;
  if (meets(mo, mc) || meets(mo, ms))
    return set_error(SIMP_RT_EINVAL, "%s: out shares memory with another operand", fn);
  BlockLaunch bl;
  if ((rc = bl.plan(fn, out_s0, s_s1))) return rc;
  const int dev = ensure_device();
  if (dev < 0) return dev;
  Operand oc, os, oo;
  if ((rc = bind_here(oc, mc.data(), mc.bytes(), Operand::kIn, dev, "codes")) ||
      (rc = bind_here(os, ms.data(), ms.bytes(), Operand::kIn, dev, "scales")) ||
      (rc = bind_here(oo, mo.data(), mo.bytes(), Operand::kOut, dev, "out")))
    return rc;
  mo.rows_of(oo);
  auto kernel = bl.run == 1 ? dequantize_mx4_k<1, false>
                : streams(oo.dev(), mo.st[0], out_s0 * out_s1) ? dequantize_mx4_k<4, true> : dequantize_mx4_k<4, false>;
  hipLaunchKernelGGL(kernel, dim3(bl.grid), dim3(256), 0, cur_stream(), (const uint8_t *)oc.dev(), mc.st[0],
                     (const uint8_t *)os.dev(), ms.st[0], (float *)oo.dev(), mo.st[0], out_s1, s_s1, bl.blocks);
  SIMP_HIP(hipGetLastError());
  Operand *ops[] = {&oc, &os, &oo};
  return finish(ops, 3);
}

int32_t simp_rt_matmul_mx4(
    const uint8_t *a_alloc, const uint8_t *a, int64_t a_off, int64_t a_s0, int64_t a_s1,
    int64_t a_st0, int64_t a_st1, const uint8_t *as_alloc, const uint8_t *a_scales, int64_t as_off,
    int64_t as_s0, int64_t as_s1, int64_t as_st0, int64_t as_st1, const uint8_t *b_alloc,
    const uint8_t *b, int64_t b_off, int64_t b_s0, int64_t b_s1, int64_t b_st0, int64_t b_st1,
    const uint8_t *bs_alloc, const uint8_t *b_scales, int64_t bs_off, int64_t bs_s0, int64_t bs_s1,
    int64_t bs_st0, int64_t bs_st1, float *out_alloc, float *out, int64_t out_off, int64_t out_s0,
    int64_t out_s1, int64_t out_st0, int64_t out_st1) {
  (void)a_alloc; (void)as_alloc; (void)b_alloc; (void)bs_alloc; (void)out_alloc;
  Mat<const uint8_t> ma{a, a_off, {a_s0, a_s1}, {a_st0, a_st1}, 0};
  Mat<const uint8_t> mas{a_scales, as_off, {as_s0, as_s1}, {as_st0, as_st1}, 0};
  Mat<const uint8_t> mb[1] = {{b, b_off, {b_s0, b_s1}, {b_st0, b_st1}, 0}};
  Mat<const uint8_t> mbs[1] = {{b_scales, bs_off, {bs_s0, bs_s1}, {bs_st0, bs_st1}, 0}};
  Mat<float> mo{out, out_off, {out_s0, out_s1}, {out_st0, out_st1}, 0};
  return product<1>("matmul_mx4", ma, mas, mb, mbs, mo);
}

int32_t simp_rt_swiglu_mx4(
    const uint8_t *a_alloc, const uint8_t *a, int64_t a_off, int64_t a_s0, int64_t a_s1,
    int64_t a_st0, int64_t a_st1, const uint8_t *as_alloc, const uint8_t *a_scales, int64_t as_off,
    int64_t as_s0, int64_t as_s1, int64_t as_st0, int64_t as_st1, const uint8_t *w1_alloc,
    const uint8_t *w1, int64_t w1_off, int64_t w1_s0, int64_t w1_s1, int64_t w1_st0, int64_t w1_st1,
    const uint8_t *s1_alloc, const uint8_t *s1, int64_t s1_off, int64_t s1_s0, int64_t s1_s1,
    int64_t s1_st0, int64_t s1_st1, const uint8_t *w3_alloc, const uint8_t *w3, int64_t w3_off,
    int64_t w3_s0, int64_t w3_s1, int64_t w3_st0, int64_t w3_st1, const uint8_t *s3_alloc,
    const uint8_t *s3, int64_t s3_off, int64_t s3_s0, int64_t s3_s1, int64_t s3_st0, int64_t s3_st1,
    float *out_alloc, float *out, int64_t out_off, int64_t out_s0, int64_t out_s1, int64_t out_st0,
    int64_t out_st1) {
  (void)a_alloc; (void)as_alloc; (void)w1_alloc; (void)s1_alloc; (void)w3_alloc; (void)s3_alloc;
  (void)out_alloc;
  Mat<const uint8_t> ma{a, a_off, {a_s0, a_s1}, {a_st0, a_st1}, 0};
  Mat<const uint8_t> mas{a_scales, as_off, {as_s0, as_s1}, {as_st0, as_st1}, 0};
  Mat<const uint8_t> mb[2] = {{w1, w1_off, {w1_s0, w1_s1}, {w1_st0, w1_st1}, 0},
                              {w3, w3_off, {w3_s0, w3_s1}, {w3_st0, w3_st1}, 0}};
  Mat<const uint8_t> mbs[2] = {{s1, s1_off, {s1_s0, s1_s1}, {s1_st0, s1_st1}, 0},
                               {s3, s3_off, {s3_s0, s3_s1}, {s3_st0, s3_st1}, 0}};
  Mat<float> mo{out, out_off, {out_s0, out_s1}, {out_st0, out_st1}, 0};
  return product<2>("swiglu_mx4", ma, mas, mb, mbs, mo);
}

}  // extern "C"
