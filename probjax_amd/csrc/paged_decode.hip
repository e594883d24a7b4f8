// Attention of each sequence's newest tokens over a paged KV cache for gfx950, in the
// cache's own type or over 8 bits:
//   o_t = sum_j softmax_j(scale q_t.k_j) v_j,  j < L - (T-1-t),
// L keys of the sequence, T new tokens (one as a rule).
//
// A workgroup per (sequence, token, query head); its waves take keys in turn, a wave
// per key, and join at the end.
#include <stdio.h>

#include "pages.h"

namespace pjx {

struct PagedArgs {
  PageArgs p;
  const char* q;
  char* o;
  float* lse;
  const int32_t* lengths;
  int B, T, Hq, D;
  float cx;
};

template <typename C, typename E>
__global__ __launch_bounds__(256) void paged_decode_simple_kernel(PagedArgs a) {
  constexpr int CS = fmt_size<C>(), ES = fmt_size<E>();
  __shared__ float red[4][256 + 2];
  const PageArgs& p = a.p;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int t = blockIdx.x / a.Hq, hq = blockIdx.x % a.Hq, b = blockIdx.y, h = hq / (a.Hq / p.H);
  const int room = p.most * p.page;
  const int L = (a.lengths ? min(max(a.lengths[b], 0), room) : room) - (a.T - 1 - t);
  const bool in = 4 * lane < a.D;
  auto load4 = [](const char* x, auto fmt, float* y) {
    typedef decltype(fmt) F;
    if constexpr (std::is_same<F, F32Fmt>::value) {
      const f32x4 r = *(const f32x4*)x;
      y[0] = r[0], y[1] = r[1], y[2] = r[2], y[3] = r[3];
    } else if constexpr (std::is_same<F, E4m3Fmt>::value) {
      const int r = *(const int*)x;
      const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(r, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(r, true);
      y[0] = lo[0], y[1] = lo[1], y[2] = hi[0], y[3] = hi[1];
    } else {
      const u32x2 r = *(const u32x2*)x;
      y[0] = F::lo(r[0]), y[1] = F::hi(r[0]), y[2] = F::lo(r[1]), y[3] = F::hi(r[1]);
    }
  };
  const int64_t row = ((int64_t)b * a.T + t) * a.Hq + hq;
  float q[4] = {}, o[4] = {}, m = kMaxInit, l = 0.f;
  if (in) load4(a.q + (row * a.D + 4 * lane) * ES, E{}, q);
  for (int j = w; j < L; j += 4) {
    const int i = p.by_page(j), slot = j - i * p.page;
    const uint32_t page = page_entry(p, b, i);
    if (page >= p.pages) continue;
    float k[4] = {}, v[4] = {};
    if (in) {
      load4(p.k + page * p.kp + slot * p.kt + h * p.kh + 4 * lane * CS, C{}, k);
      load4(p.v + page * p.vp + slot * p.vt + h * p.vh + 4 * lane * CS, C{}, v);
    }
    float s = (q[0] * k[0] + q[1] * k[1]) + (q[2] * k[2] + q[3] * k[3]);
    for (int x = 32; x; x >>= 1) s += __shfl_xor(s, x);
    float vs = 1.f;
    if constexpr (CS == 1) {
      const int64_t e = ((int64_t)page * p.H + h) * p.page + slot;
      s *= exponent_scale(p.ke[e]);
      vs = exponent_scale(p.ve[e]);
    }
    s *= a.cx;
    const float mn = fmaxf(m, s), corr = fast_exp2(m - mn), pr = fast_exp2(s - mn);
    m = mn;
    l = fmaf(l, corr, pr);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(o[e], corr, pr * vs * v[e]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) red[w][4 * lane + e] = o[e];
  if (lane == 0) red[w][256] = m, red[w][257] = l;
  __syncthreads();
  if (w) return;
  float M = kMaxInit, den = 0.f, sum[4] = {};
  for (int x = 0; x < 4; ++x) M = fmaxf(M, red[x][256]);
  for (int x = 0; x < 4; ++x) {
    const float f = fast_exp2(red[x][256] - M);
    den = fmaf(red[x][257], f, den);
    for (int e = 0; e < 4; ++e) sum[e] = fmaf(red[x][4 * lane + e], f, sum[e]);
  }
  uint32_t bits = __float_as_uint(den);
  asm volatile("" : "+v"(bits));  // (compiled without NaN in mind: a NaN sum is one of some key)
  const bool some = bits != 0u;
  float out[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = some ? sum[e] / den : 0.f;
  if (in) {
    char* to = a.o + (row * a.D + 4 * lane) * ES;
    if constexpr (ES == 4) *(f32x4*)to = f32x4{out[0], out[1], out[2], out[3]};
    else *(u32x2*)to = u32x2{E::pack2(out[0], out[1]), E::pack2(out[2], out[3])};
  }
  if (a.lse && lane == 0) a.lse[((int64_t)b * a.Hq + hq) * a.T + t] = some ? (M + __log2f(den)) * kLn2 : INFINITY;
}

template <typename C, typename E>
static int run_simple(const PagedArgs& a, hipStream_t s, const char* who) {
  launch_kernel<paged_decode_simple_kernel<C, E>>(dim3((unsigned)(a.Hq * a.T), (unsigned)a.B), dim3(256), 0, s, a);
  return check_launch(who);
}

}  // namespace pjx

using namespace pjx;

extern "C" size_t pjx_paged_decode_workspace_size(int64_t, int64_t, int64_t, int64_t, int64_t) { return 16; }

extern "C" int pjx_paged_decode(int dtype, int cache_dtype, const void* q, const pjx_pages* cache,
                                const int32_t* kv_lengths, void* o, float* lse, void* workspace,
                                size_t workspace_bytes, int64_t batch, int64_t q_len, int64_t q_heads,
                                int64_t kv_heads, int64_t head_dim, float sm_scale, void* stream) {
  clear_error();
  const char* who = "pjx_paged_decode";
  PagedArgs a = {};
  const int rc = fill_pages(a.p, who, cache_dtype, cache, batch, kv_heads, head_dim);
  if (rc != PJX_OK) return rc;
  if (dtype != PJX_DTYPE_BF16 && dtype != PJX_DTYPE_F16 && dtype != PJX_DTYPE_F32)
    return fail(PJX_ERR_INVALID, "pjx_paged_decode: dtype must be PJX_DTYPE_BF16, PJX_DTYPE_F16 or PJX_DTYPE_F32");
  const bool quant = cache_dtype == PJX_DTYPE_E4M3;
  if (!quant && cache_dtype != dtype) return fail(PJX_ERR_INVALID, "pjx_paged_decode: the cache has another dtype");
  if (q_len <= 0 || q_heads <= 0 || q_heads % kv_heads) return fail(PJX_ERR_INVALID, "pjx_paged_decode: bad sizes");
  if (q_len > (1 << 20) || q_heads > (1 << 20) || batch * q_heads > (1 << 30) || batch * q_heads * q_len > (1 << 30))
    return fail(PJX_ERR_INVALID, "pjx_paged_decode: sizes out of range");
  if (!(sm_scale > 0.f)) return fail(PJX_ERR_INVALID, "pjx_paged_decode: sm_scale must be > 0");
  if (batch == 0) return PJX_OK;
  if (!q || !o) return fail(PJX_ERR_INVALID, "pjx_paged_decode: null pointer");
  if (((uintptr_t)q | (uintptr_t)o) % 16) return fail(PJX_ERR_INVALID, "pjx_paged_decode: q and o must start on 16 bytes");
  if (!workspace || workspace_bytes < 16) return fail(PJX_ERR_WORKSPACE, "pjx_paged_decode: workspace missing or too small");
  a.q = (const char*)q; a.o = (char*)o; a.lse = lse; a.lengths = kv_lengths;
  a.B = (int)batch; a.T = (int)q_len; a.Hq = (int)q_heads; a.D = (int)head_dim;
  a.cx = sm_scale * kLog2e;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == PJX_DTYPE_F32)
    return quant ? run_simple<E4m3Fmt, F32Fmt>(a, s, who) : run_simple<F32Fmt, F32Fmt>(a, s, who);
  if (dtype == PJX_DTYPE_BF16)
    return quant ? run_simple<E4m3Fmt, Bf16Fmt>(a, s, who) : run_simple<Bf16Fmt, Bf16Fmt>(a, s, who);
  return quant ? run_simple<E4m3Fmt, F16Fmt>(a, s, who) : run_simple<F16Fmt, F16Fmt>(a, s, who);
}
