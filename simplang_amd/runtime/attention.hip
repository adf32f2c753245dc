// attention.hip -- causal attention of packed prompts (simp_rt_attention_packed_f32).
//
// out_i = sum_j p_ij v_j, p_i = softmax_j(scale q_i . k_j) over the keys j <= i +
// nk - nq of the row's sequence.  One pass over the keys with a running maximum m
// and sum l: o and l are scaled by e^(m_old - m_new) when a tile raises m.
#include <cmath>

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

// The fp32 MFMA form.  A block takes 16 queries of one head; its four waves take the
// 16-key tiles in turn, each with its own running maximum, sum and output,
// combined through LDS at the end.  S^T = K Q^T on v_mfma_f32_16x16x4_f32 leaves a
// lane with the scores of keys 4g .. 4g+3 (g = lane / 16) for query lane % 16, the
// B operand of O^T += V^T P^T.  HB: 16-dimension blocks of a head.  VEC: rows are
// whole 16-byte chunks (head_size and strides multiples of 4, aligned pointers).
template <int HB, bool VEC>
__global__ void __launch_bounds__(256) attn_packed_f32_k(const PackedArgs a) {
  __shared__ float so[4][16 * HB][17];
  __shared__ float sm[4][16], sl[4][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int r16 = lane & 15, g = lane >> 4, hs = a.hs;
  const int t = (int)(gridDim.x - 1 - blockIdx.x), h = blockIdx.y;
  const int s = seq_of_slot<16>(a.q_starts, a.n, a.tq, t);
  const int qb = clampi(a.q_starts[s], 0, a.tq), qe = clampi(a.q_starts[s + 1], qb, a.tq);
  const int kb = clampi(a.k_starts[s], 0, a.tk), ke = clampi(a.k_starts[s + 1], kb, a.tk);
  const int nq = qe - qb, nk = ke - kb;
  const int slot0 = qb / 16 + s;
  if (t < slot0 || t - slot0 >= (nq + 15) / 16) return;
  const int q0 = 16 * (t - slot0);
  const int my = min(q0 + r16, nq - 1) + nk - nq;              // the lane's last key, or negative
  const int last = min(q0 + 15, nq - 1) + nk - nq;             // the block's
  const float *kp = a.k + (int64_t)kb * a.k_row + (h / a.group) * a.k_head;
  const float *vp = a.v + (int64_t)kb * a.v_row + (h / a.group) * a.v_head;

  auto load4 = [&](const float *row, int d) {
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
  };
  float4 q[HB];
  {
    const float *qr = a.q + (int64_t)(qb + min(q0 + r16, nq - 1)) * a.q_row + h * a.q_head;
#pragma unroll
    for (int j = 0; j < HB; j++) q[j] = load4(qr, 16 * j + 4 * g);
  }
  v4f o[HB];
#pragma unroll
  for (int j = 0; j < HB; j++) o[j] = v4f{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  for (int key0 = 16 * wave; key0 <= last; key0 += 64) {
    float v[HB][4];  // V[key0 + 4g + r][16 j + r16]
    v4f sc = {0.f, 0.f, 0.f, 0.f};
    {
      const float *kr = kp + (int64_t)min(key0 + r16, last) * a.k_row;
#pragma unroll
      for (int j = 0; j < HB; j++) {
        const float4 k = load4(kr, 16 * j + 4 * g);
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
    if (key0 + 15 > q0 + nk - nq && __any(odd)) {
      // Some query does not see all 16 keys, and a product with a hidden infinity
      // or NaN would reach its row: one key at a time, added where it is seen.
      for (int kk = 0; kk < 16; kk++) {
        const int src = (kk >> 2) * 16 + r16;
        const float pr = kk & 2 ? (kk & 1 ? p[3] : p[2]) : (kk & 1 ? p[1] : p[0]);
        const float pk = __shfl(pr, src);
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
  {
    float x = l, y = l;
    permlane16_swap(x, y);
    l = x + y;
    x = y = l;
    permlane32_swap(x, y);
    l = x + y;
  }
  if (g == 0) {
    sm[wave][r16] = m;
    sl[wave][r16] = l;
  }
#pragma unroll
  for (int j = 0; j < HB; j++)
#pragma unroll
    for (int r = 0; r < 4; r++) so[wave][16 * j + 4 * g + r][r16] = o[j][r];
  __syncthreads();
  for (int e = threadIdx.x; e < 16 * hs; e += 256) {
    const int qi = e / hs, d = e - qi * hs;
    if (q0 + qi >= nq) break;  // queries in increasing order
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) M = fmaxf(M, sm[w][qi]);
    const float mu = M == -INFINITY ? 0.f : M;
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float f = expf(sm[w][qi] - mu);
      num = fmaf(f, so[w][d][qi], num);
      den = fmaf(f, sl[w][qi], den);
    }
    const bool none = q0 + qi + nk - nq < 0;
    a.out[(int64_t)(qb + q0 + qi) * a.o_row + h * a.o_head + d] = none ? 0.f : num / den;
  }
}

template <bool VEC>
void launch_f32(const PackedArgs &a, dim3 grid, hipStream_t st) {
#define ATTN(HB) hipLaunchKernelGGL((attn_packed_f32_k<HB, VEC>), grid, dim3(256), 0, st, a)
  if (a.hs <= 32) ATTN(2);
  else if (a.hs <= 64) ATTN(4);
  else if (a.hs <= 128) ATTN(8);
  else ATTN(16);
#undef ATTN
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
  const bool vec = a.hs % 4 == 0 && ((q_st0 | q_st1 | k_st0 | k_st1) & 3) == 0 &&
                   (((uintptr_t)a.q | (uintptr_t)a.k) & 15) == 0;
  const dim3 grid((unsigned)(q_s0 / 16 + n), (unsigned)q_s1);
  if (vec) launch_f32<true>(a, grid, cur_stream());
  else launch_f32<false>(a, grid, cur_stream());
  Operand *ops[] = {&oq, &ok, &ov, &oo, &oqs, &oks};
  return finish(ops, 6);
}

}  // extern "C"
