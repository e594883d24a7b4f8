// Attention of drafted tokens over a KV cache for gfx950.  A draft of T tokens
// forms a tree: token t continues token parents[t], or the sequence itself.
// Their keys lie in the cache behind the sequence's prefix, and token t sees
// the prefix, itself and the tokens it descends from:
//   o_t = sum_j softmax_j(scale q_t.k_j) v_j,  j in [0, P) or P + anc(t).
//
// It is the split-KV decode (decode_common.h) with (Hq/Hkv)*T packed query
// rows, plus a table of what each token sees, which a work item builds in LDS
// if its keys reach past the prefix and asks on the 32-key steps that do; the
// steps over the prefix are the decode's.  These kernels take up to 32 rows per KV
// head in 16 bits (more: tree_wide.hip) and any number of float32 ones.  Bound by
// latency on small caches (2 x 512 float32 keys, 5 tokens of 4 heads of 64: 7.2 us and
// 3 for the merge; 4 bf16 tokens over 4096 keys, 8 KV heads of 128: 13.4 us for both)
// and in float32 by a work item's phases, which two workgroups per CU overlap: 8 x
// 4096 keys, 32 rows of 128, 67 MB: 28 us.
#include <stdio.h>

#include "decode_common.h"

namespace pjx {

template <typename E, int D, int NRB, bool ROWS>
__global__ __launch_bounds__(256, (decode_occupancy<D, D, NRB>())) void tree_decode_kernel(DecodeArgs a) {
  gqa_decode<E, D, D, NRB, false, ROWS, kTree>(a);
}

template <int D, int NRB>
__global__ __launch_bounds__(256, 1) void tree_decode_f32_kernel(DecodeArgs a) {
  gqa_decode_f32<D, D, NRB, kTree>(a);
}

template <typename E, int D, bool ROWS>
static int run_tree_rows(DecodeArgs& a, int nrb, void* ws, size_t ws_bytes, hipStream_t s, const char* who) {
  if (nrb == 1) return run_decode<tree_decode_kernel<E, D, 1, ROWS>>(a, ws, ws_bytes, s, who);
  if (nrb == 2) return run_decode<tree_decode_kernel<E, D, 2, ROWS>>(a, ws, ws_bytes, s, who);
  return fail(PJX_ERR_INVALID, "tree decode: row blocks");
}

template <typename E>
static int run_tree(DecodeArgs& a, int d, int nrb, void* ws, size_t ws_bytes, hipStream_t s, const char* who) {
  const bool rows = a.orow != d;
  if (d == 64)
    return rows ? run_tree_rows<E, 64, true>(a, nrb, ws, ws_bytes, s, who)
                : run_tree_rows<E, 64, false>(a, nrb, ws, ws_bytes, s, who);
  if (d == 128)
    return rows ? run_tree_rows<E, 128, true>(a, nrb, ws, ws_bytes, s, who)
                : run_tree_rows<E, 128, false>(a, nrb, ws, ws_bytes, s, who);
  return run_tree_rows<E, 256, false>(a, nrb, ws, ws_bytes, s, who);
}

template <int D>
static int run_tree_f32(DecodeArgs& a, int nrb, void* ws, size_t ws_bytes, hipStream_t s, const char* who) {
  // (heads of 256: 32 rows spill registers, 47 us for 39 on 2 x 2048 keys of 8 heads, 20 tokens)
  if constexpr (D <= 128)
    if (nrb > 1) return run_decode<tree_decode_f32_kernel<D, 2>>(a, ws, ws_bytes, s, who);
  return run_decode<tree_decode_f32_kernel<D, 1>>(a, ws, ws_bytes, s, who);
}

// Argument checks shared by the decode forms of this library's cache operators:
// sizes, head dim / row width, alignment, strides; resolves chunk = 0 and fills
// the decode arguments.
int fill_cache_decode(DecodeArgs& a, const char* who, int dtype, const void* q, const void* k, const void* v,
                      const int32_t* kv_lengths, void* o, float* lse, int64_t batch, int64_t q_len, int64_t kv_len,
                      int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t row_dim,
                      const pjx_cache_strides* strides, float sm_scale, int64_t chunk) {
  char buf[256];
  auto bad = [&](const char* what) {
    snprintf(buf, sizeof(buf), "%s: %s", who, what);
    return fail(PJX_ERR_INVALID, buf);
  };
  if (dtype != PJX_DTYPE_BF16 && dtype != PJX_DTYPE_F16 && dtype != PJX_DTYPE_F32)
    return bad("dtype must be PJX_DTYPE_BF16, PJX_DTYPE_F16 or PJX_DTYPE_F32");
  if (batch < 0 || q_len <= 0 || kv_len < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads)
    return bad("bad sizes");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return bad("head_dim must be 64, 128 or 256");
  const bool f32 = dtype == PJX_DTYPE_F32;
  if (row_dim != head_dim && (f32 || head_dim == 256 || row_dim <= 0 || row_dim > head_dim || row_dim % 8))
    return bad("row_dim must be head_dim, or in 16 bits a multiple of 8 up to a head_dim of 64 or 128");
  if (!(sm_scale > 0.f)) return bad("sm_scale must be > 0");
  if (chunk == 0) chunk = auto_chunk(batch, kv_heads, kv_len, kGqaItems);
  if (chunk < 128 || chunk % 128) return bad("chunk must be a positive multiple of 128");
  const int64_t rows = (q_heads / kv_heads) * q_len, most = (int64_t)1 << 40;
  if (kv_len > (1 << 30) || rows > (1 << 20) || batch > (1 << 24) || kv_heads > (1 << 24) ||
      batch * q_heads > (1 << 30) || batch * q_heads * q_len > (1 << 30) || batch * q_heads * q_len * head_dim > most ||
      batch * kv_heads > most / head_dim / std::max<int64_t>(kv_len, 1))
    return bad("sizes out of range");
  if (batch == 0) return PJX_OK;
  if (!q || !o || (kv_len > 0 && (!k || !v))) return bad("null pointer");
  const int64_t cache_row = kv_heads * row_dim;
  a = {};
  a.k_b = a.v_b = kv_len * cache_row;
  a.k_t = a.v_t = cache_row;
  a.k_h = a.v_h = row_dim;
  if (strides) {
    const int64_t s[6] = {strides->k_batch, strides->k_token, strides->k_head,
                          strides->v_batch, strides->v_token, strides->v_head};
    for (int64_t x : s) {
      if (x < 0 || x > most) return bad("cache strides out of range");
      if (x % (f32 ? 4 : 8)) return bad("cache strides must be whole 16-byte chunks");
    }
    a.k_b = s[0]; a.k_t = s[1]; a.k_h = s[2];
    a.v_b = s[3]; a.v_t = s[4]; a.v_h = s[5];
  }
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)o) % 16) return bad("q, k, v and o must start on 16 bytes");
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
  a.lengths = kv_lengths; a.lse = lse;
  if (f32) a.o32 = (float*)o;
  else a.o = (uint16_t*)o;
  a.f16 = dtype == PJX_DTYPE_F16;
  a.B = (int)batch; a.Lq = (int)q_len; a.Lk = (int)kv_len; a.Hq = (int)q_heads; a.G = (int)kv_heads;
  a.rows = (int)rows; a.chunk = (int)chunk;
  a.nch = (int)std::max<int64_t>((kv_len + chunk - 1) / chunk, 1);
  a.dv = (int)head_dim; a.orow = (int)row_dim; a.cx = sm_scale * kLog2e;
  return PJX_OK;
}

}  // namespace pjx

using namespace pjx;

extern "C" int pjx_tree_decode(int dtype, const void* q, const void* k, const void* v, const int32_t* kv_lengths,
                               const int32_t* parents, const uint8_t* tree_mask, int64_t trees, void* o, float* lse,
                               void* workspace, size_t workspace_bytes, int64_t batch, int64_t q_len, int64_t kv_len,
                               int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t row_dim,
                               const pjx_cache_strides* strides, float sm_scale, int64_t chunk, void* stream) {
  clear_error();
  const char* who = "pjx_tree_decode";
  DecodeArgs a = {};
  const int rc = fill_cache_decode(a, who, dtype, q, k, v, kv_lengths, o, lse, batch, q_len, kv_len, q_heads, kv_heads,
                                   head_dim, row_dim, strides, sm_scale, chunk);
  if (rc != PJX_OK) return rc;
  if (q_len > kTreeMax) return fail(PJX_ERR_INVALID, "pjx_tree_decode: at most 256 drafted tokens");
  if (!parents == !tree_mask) return fail(PJX_ERR_INVALID, "pjx_tree_decode: parents or tree_mask, and not both");
  if (trees != 1 && trees != batch) return fail(PJX_ERR_INVALID, "pjx_tree_decode: one tree, or one per sequence");
  if (!kv_lengths && kv_len < q_len)
    return fail(PJX_ERR_INVALID, "pjx_tree_decode: without kv_lengths the cache must hold the drafted tokens' keys");
  if (batch == 0) return PJX_OK;
  hipStream_t s = (hipStream_t)stream;
  const bool f32 = dtype == PJX_DTYPE_F32;
  if (kv_len == 0)
    return write_keyless(o, lse, (size_t)(batch * q_len * q_heads * row_dim), f32, (size_t)(batch * q_heads * q_len), s,
                         who);
  a.extra = (int)q_len;
  a.parents = parents;
  a.tree_mask = tree_mask;
  a.tree_step = trees == 1 ? 0 : parents ? q_len : q_len * q_len;
  const int d = (int)head_dim;
  if (tree_wide_takes(a, d, f32)) return run_tree_wide(a, d, chunk == 0, workspace, workspace_bytes, s, who);
  // (at most 32 rows, or rows too far apart in memory for the wide kernel)
  const int nrb = std::min(gqa_row_blocks(a.rows, d, d, f32), f32 && d == 256 ? 1 : 2);
  a.rpg = kRows * nrb;
  if (f32)
    return d == 64    ? run_tree_f32<64>(a, nrb, workspace, workspace_bytes, s, who)
           : d == 128 ? run_tree_f32<128>(a, nrb, workspace, workspace_bytes, s, who)
                      : run_tree_f32<256>(a, nrb, workspace, workspace_bytes, s, who);
  return a.f16 ? run_tree<F16Fmt>(a, d, nrb, workspace, workspace_bytes, s, who)
               : run_tree<Bf16Fmt>(a, d, nrb, workspace, workspace_bytes, s, who);
}
