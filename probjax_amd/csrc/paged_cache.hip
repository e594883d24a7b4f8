// Writing to and reading from a paged KV cache for gfx950, the cache in the type of
// its keys or in 8 bits.
//
// In 8 bits every row x (one token's key or value of one head) is held as e4m3 codes c
// and one exponent e:  e = the least integer with max|x| <= 448 * 2^e, c = e4m3(x 2^-e),
// read back as c 2^e.  A power of two makes the division exact, so a value is rounded
// once, to the nearest of the type's 4 significant bits (at most 2^-4 of it), down to
// 2^-13 of the row's largest; below that e4m3's steps are even.  Finer blocks or scales
// of more bits would not change those 4 bits.
//
// Both kernels move every byte once and are bound by HBM: a group of lanes per row, 16
// bytes of the 16-bit or float32 side a lane, several rows of a thread in flight.  8 heads
// of 128: 8 x 300-4096 new keys from bf16 to 8 bits 108 MB in 23 us (4.7 TB/s), one key of
// 32 sequences 3.3; 4 x 2048 keys of 4 heads of 256 copied, 67 MB in 12 (5.4).  Read back,
// 16 x 1000-8192 keys from 8 bits to bf16 689 MB in 132 (5.2).  A large copy reaches 5.1.
#include <stdio.h>

#include "pages.h"

namespace pjx {

constexpr int kPageThreads = 256;

struct WriteArgs {
  PageArgs p;
  const char* x[2];  // new k, v
  int64_t xb[2], xt[2], xh[2];  // bytes
  const int32_t *lengths, *fresh;
  int32_t* lengths_out;
  int B, T, D;
  int tokens;  // of a workgroup
  FastDiv by_h;
};

// Keys of sequence b before the call, and its new tokens.
__device__ __forceinline__ void new_tokens(const WriteArgs& a, int b, int64_t& before, int& n) {
  before = a.lengths ? max(a.lengths[b], 0) : 0;
  n = a.fresh ? min(max(a.fresh[b], 0), a.T) : a.T;
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t x) {
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true));
}
// Largest of a group of LPR lanes (8, 16 or 32), in all of them.
template <int LPR>
__device__ __forceinline__ uint32_t group_max(uint32_t x) {
  x = dpp_max<0xb1>(x);   // lane ^ 1
  x = dpp_max<0x4e>(x);   // lane ^ 2
  x = dpp_max<0x141>(x);  // the other half of 8
  if constexpr (LPR >= 16) x = dpp_max<0x140>(x);  // the other half of 16
  if constexpr (LPR >= 32) {
    auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max((uint32_t)r[0], (uint32_t)r[1]);
  }
  return x;
}

// What 8 elements of a row in format E are made of.
template <typename E>
struct Row8 {
  static constexpr bool k32 = std::is_same<E, F32Fmt>::value, kF16 = std::is_same<E, F16Fmt>::value;
  // The largest magnitude that reads back inside the type's range is 240 * 2^e, of those
  // below 256 * 2^e: past it a row takes the long way.  (As the type's own bits; infinities
  // and NaN are past it too.  Bits, since the sources are compiled without NaN in mind.)
  static constexpr uint32_t kMost = k32 ? 0x7f700000u : kF16 ? 0x7b80u : 0x7f70u;
  static constexpr uint32_t kInf = k32 ? 0x7f800000u : kF16 ? 0x7c00u : 0x7f80u;

  __device__ __forceinline__ static uint32_t magnitude(const u32x4* raw, int i) {
    if constexpr (k32) return raw[i / 4][i % 4] & 0x7fffffffu;
    else return (raw[0][i / 2] >> 16 * (i % 2)) & 0x7fffu;
  }
  __device__ __forceinline__ static float value(const u32x4* raw, int i) {
    if constexpr (k32) return __uint_as_float(raw[i / 4][i % 4]);
    else return i % 2 ? E::hi(raw[0][i / 2]) : E::lo(raw[0][i / 2]);
  }
  __device__ __forceinline__ static uint32_t float_bits(uint32_t m) {  // of a magnitude
    if constexpr (k32) return m;
    else return __float_as_uint(E::lo(m));
  }
  __device__ __forceinline__ static uint32_t largest(const u32x4* raw) {
    uint32_t m = 0;
    if constexpr (k32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, magnitude(raw, i));
    } else {  // two at a time
      typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
      u16x2 x = __builtin_bit_cast(u16x2, raw[0][0] & 0x7fff7fffu);
#pragma unroll
      for (int i = 1; i < 4; ++i) x = __builtin_elementwise_max(x, __builtin_bit_cast(u16x2, raw[0][i] & 0x7fff7fffu));
      m = max((uint32_t)x[0], (uint32_t)x[1]);
    }
    return m;
  }
};

// The exponent byte of a row whose largest finite value has these float bits: 448 is 1.75 *
// 2^8, its fraction's bits 0x600000; a scale below 2^-126 would be subnormal.
__device__ __forceinline__ int row_exponent(uint32_t bits) {
  return max((int)(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), 1);
}

// E: format of the new rows.  QUANT: into 8 bits, 8 elements a lane; else copied, 16
// bytes a lane.  LPR lanes per row.
template <typename E, bool QUANT, int LPR>
__global__ __launch_bounds__(kPageThreads) void write_pages_kernel(WriteArgs a) {
  typedef Row8<E> R;
  constexpr int SZ = fmt_size<E>();
  constexpr int EPL = QUANT ? 8 : 16 / SZ;  // elements of a lane
  constexpr int LDS16 = EPL * SZ / 16;      // its 16-byte loads
  constexpr int RPB = kPageThreads / LPR;   // rows of a pass
  constexpr int U = 4;                      // passes in flight
  const PageArgs& p = a.p;
  const int tid = threadIdx.x, sub = tid % LPR, kv = blockIdx.z;
  const bool in_row = sub * EPL < a.D;
  char* pool = kv ? p.v : p.k;
  uint8_t* exps = kv ? p.ve : p.ke;
  const int64_t sp = kv ? p.vp : p.kp, st = kv ? p.vt : p.kt, sh = kv ? p.vh : p.kh;
  const int64_t xt = a.xt[kv], xh = a.xh[kv];
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    int64_t before;
    int n;
    new_tokens(a, b, before, n);
    const int64_t room = (int64_t)p.most * p.page;
    if (blockIdx.x == 0 && kv == 0 && tid == 0) a.lengths_out[b] = (int32_t)min(before + n, room);
    const int64_t first = (int64_t)blockIdx.x * a.tokens;
    if (first >= n || before + first >= room) continue;
    const int nt = (int)min((int64_t)a.tokens, min((int64_t)n - first, room - before - first));
    const int rows = nt * p.H;
    const char* x = a.x[kv] + b * a.xb[kv] + first * xt + sub * EPL * SZ;
    for (int r0 = 0; r0 < rows; r0 += U * RPB) {
      u32x4 raw[U][LDS16];
      uint32_t page[U];
      int slot[U], h[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r0 + u * RPB >= rows) break;
        const int mine = r0 + u * RPB + tid / LPR, r = min(mine, rows - 1), t = a.by_h(r);
        h[u] = r - t * p.H;
        const int pos = (int)(before + first) + t, i = p.by_page(pos);
        slot[u] = pos - i * p.page;
        page[u] = mine < rows ? page_entry(p, b, i) : ~0u;
#pragma unroll
        for (int j = 0; j < LDS16; ++j)
          raw[u][j] = in_row ? *(const u32x4*)(x + t * xt + h[u] * xh + 16 * j) : u32x4{0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (r0 + u * RPB >= rows) break;
        const bool there = page[u] < p.pages;
        char* to = pool + page[u] * (uint64_t)sp + slot[u] * st + h[u] * sh;
        if constexpr (QUANT) {
          uint32_t m = group_max<LPR>(R::largest(raw[u]));
          int e = row_exponent(R::float_bits(m));
          float back = exponent_scale(254 - e);
          u32x2 c;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            int w = __builtin_amdgcn_cvt_pk_fp8_f32(R::value(raw[u], 4 * i) * back, R::value(raw[u], 4 * i + 1) * back, 0, false);
            c[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(R::value(raw[u], 4 * i + 2) * back,
                                                             R::value(raw[u], 4 * i + 3) * back, w, true);
          }
          if (m > R::kMost) {
            m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t y = R::magnitude(raw[u], i);
              m = max(m, y < R::kInf ? y : 0u);
            }
            m = group_max<LPR>(m);
            e = row_exponent(R::float_bits(m));
            back = exponent_scale(254 - e);
            const float most = __uint_as_float(R::float_bits(R::kMost));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float y = fminf(fmaxf(R::value(raw[u], i), -most), most) * back;
              const uint32_t code = R::magnitude(raw[u], i) < R::kInf ? (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xffu : 0x7fu;
              c[i / 4] = (c[i / 4] & ~(0xffu << 8 * (i % 4))) | code << 8 * (i % 4);
            }
          }
          if (there) {
            // (past the caches' reuse hint: 108 MB moved in 23 us against 27)
            if (in_row) __builtin_nontemporal_store(c, (u32x2*)(to + sub * EPL));
            if (sub == 0) exps[((int64_t)page[u] * p.H + h[u]) * p.page + slot[u]] = (uint8_t)e;
          }
        } else if (there && in_row) {
          *(u32x4*)(to + sub * 16) = raw[u][0];
        }
      }
    }
  }
}

struct ReadArgs {
  PageArgs p;
  const int32_t* lengths;
  char* y[2];
  int B, D;
  int64_t L;   // tokens written of every sequence
  int tokens;  // of a workgroup
  int upr;     // 16-byte units of an output row
  FastDiv by_token, by_row;  // units of a token (H rows), of a row
};

// C: format of the cache, E: of the output (C, unless C is e4m3).  STREAM: more than the
// 256 MB cache holds, past its reuse hint and twice the rows in flight (16 x 1000-8192 keys
// of 8 heads of 128 from 8 bits, 545 MB written: 134 us against 162; 134 MB: 45 and 46, 67
// MB: 27 and 19).
template <typename C, typename E, bool STREAM>
__global__ __launch_bounds__(kPageThreads) void read_pages_kernel(ReadArgs a) {
  constexpr bool QUANT = std::is_same<C, E4m3Fmt>::value;
  constexpr int EPU = 16 / fmt_size<E>();         // elements of a unit
  constexpr int IN = EPU * fmt_size<C>();         // its bytes in the cache
  constexpr int U = STREAM ? 8 : 4;
  typedef typename std::conditional<IN == 16, u32x4, typename std::conditional<IN == 8, u32x2, uint32_t>::type>::type Raw;
  const PageArgs& p = a.p;
  const int tid = threadIdx.x, kv = blockIdx.z;
  const int64_t first = (int64_t)blockIdx.x * a.tokens;
  const int nt = (int)min((int64_t)a.tokens, a.L - first);
  const int per_token = p.H * a.upr, units = nt * per_token;
  const char* pool = kv ? p.v : p.k;
  const uint8_t* exps = kv ? p.ve : p.ke;
  const int64_t sp = kv ? p.vp : p.kp, st = kv ? p.vt : p.kt, sh = kv ? p.vh : p.kh;
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    const int64_t room = (int64_t)p.most * p.page;
    const int64_t len = a.lengths ? min((int64_t)max(a.lengths[b], 0), room) : room;
    char* y = a.y[kv] + ((int64_t)b * a.L + first) * per_token * 16;
    for (int u0 = tid; u0 < units; u0 += U * kPageThreads) {
      Raw raw[U];
      uint32_t e[U];
      bool there[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int unit = u0 + u * kPageThreads;
        const bool ok = unit < units;
        const int t = a.by_token(ok ? unit : 0), rest = (ok ? unit : 0) - t * per_token;
        const int h = a.by_row(rest), c = rest - h * a.upr;
        there[u] = ok && first + t < len;
        raw[u] = Raw{};
        e[u] = 0;
        if (there[u]) {
          const int pos = (int)first + t, i = p.by_page(pos), slot = pos - i * p.page;
          const uint32_t page = page_entry(p, b, i);
          there[u] = page < p.pages;
          if (there[u]) {
            const Raw* x = (const Raw*)(pool + page * sp + slot * st + h * sh + c * IN);
            if constexpr (STREAM) raw[u] = __builtin_nontemporal_load(x);
            else raw[u] = *x;
            if constexpr (QUANT) e[u] = exps[((int64_t)page * p.H + h) * p.page + slot];
          }
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int unit = u0 + u * kPageThreads;
        if (unit >= units) continue;
        u32x4 out = {0u, 0u, 0u, 0u};
        if constexpr (!QUANT) {
          out = raw[u];
        } else {
          const float scale = exponent_scale(e[u]);
          float x[EPU];
#pragma unroll
          for (int i = 0; i < EPU; i += 4) {
            uint32_t w;
            if constexpr (IN == 8) w = raw[u][i / 4];
            else w = raw[u];
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
            x[i] = lo[0] * scale, x[i + 1] = lo[1] * scale, x[i + 2] = hi[0] * scale, x[i + 3] = hi[1] * scale;
          }
          if constexpr (EPU == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = __float_as_uint(x[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = E::pack2(x[2 * i], x[2 * i + 1]);
          }
          if (!there[u]) out = u32x4{0u, 0u, 0u, 0u};
        }
        u32x4* to = (u32x4*)(y + (int64_t)unit * 16);
        if constexpr (STREAM) __builtin_nontemporal_store(out, to);
        else *to = out;
      }
    }
  }
}

int fill_pages(PageArgs& a, const char* who, int cache_dtype, const pjx_pages* c, int64_t batch, int64_t kv_heads,
               int64_t head_dim) {
  char buf[256];
  auto bad = [&](const char* what) {
    snprintf(buf, sizeof(buf), "%s: %s", who, what);
    return fail(PJX_ERR_INVALID, buf);
  };
  const bool e4m3 = cache_dtype == PJX_DTYPE_E4M3, f32 = cache_dtype == PJX_DTYPE_F32;
  if (!e4m3 && !f32 && cache_dtype != PJX_DTYPE_BF16 && cache_dtype != PJX_DTYPE_F16)
    return bad("cache_dtype must be PJX_DTYPE_F32, PJX_DTYPE_BF16, PJX_DTYPE_F16 or PJX_DTYPE_E4M3");
  if (!c) return bad("null cache");
  const int64_t size = e4m3 ? 1 : f32 ? 4 : 2, most = (int64_t)1 << 40;
  if (batch < 0 || kv_heads <= 0 || c->pages < 0 || c->page_size <= 0 || c->table_len < 0) return bad("bad sizes");
  if (head_dim <= 0 || head_dim > 256 || head_dim * size % 16)
    return bad("head_dim must be at most 256 and a row of the cache whole 16-byte chunks");
  if (batch > (1 << 24) || kv_heads > (1 << 20) || c->pages > 0x7fffffffLL || c->page_size > (1 << 30) ||
      c->table_len > (1 << 30) || c->page_size * c->table_len > (1 << 30))
    return bad("sizes out of range (a sequence holds at most 2^30 keys)");
  if (!c->table && batch > 0 && c->table_len > 0 && (c->table_len > 1 || c->pages < batch))
    return bad("without a table every sequence has the page of its number");
  if (c->table && (c->table_stride < 0 || c->table_stride > most)) return bad("table stride out of range");
  const int64_t s[6] = {c->k_page, c->k_token, c->k_head, c->v_page, c->v_token, c->v_head};
  for (int64_t x : s) {
    if (x < 0 || x > most) return bad("cache strides out of range");
    if (x * size % 16) return bad("cache strides must be whole 16-byte chunks");
  }
  if (batch > 0 && c->pages > 0 && c->table_len > 0) {
    if (!c->k || !c->v || (e4m3 && (!c->k_exponents || !c->v_exponents))) return bad("null pointer");
    if (((uintptr_t)c->k | (uintptr_t)c->v) % 16) return bad("the cache must start on 16 bytes");
  }
  a = {};
  a.k = (char*)c->k; a.v = (char*)c->v;
  a.ke = (uint8_t*)c->k_exponents; a.ve = (uint8_t*)c->v_exponents;
  a.table = c->table;
  a.table_step = c->table_stride;
  a.pages = (uint32_t)c->pages;
  a.page = (int)c->page_size;
  a.most = (int)c->table_len;
  a.H = (int)kv_heads;
  a.by_page = fast_div(c->page_size);
  a.kp = s[0] * size; a.kt = s[1] * size; a.kh = s[2] * size;
  a.vp = s[3] * size; a.vt = s[4] * size; a.vh = s[5] * size;
  return PJX_OK;
}

constexpr int64_t kStreamRead = (int64_t)256 << 20;  // bytes read_pages writes past which they are streamed

// Tokens of a workgroup whose tokens are `per_token` units of work, `passes` x 256 of
// them wanted.
static int tokens_of(int64_t per_token, int passes) {
  return (int)std::max<int64_t>((int64_t)passes * kPageThreads / per_token, 1);
}

// Whether a launch's 32 bits count the threads of so many workgroups.
static bool countable(int64_t workgroups) { return workgroups * kPageThreads <= 0xffffffffLL; }

template <typename E, bool QUANT, int LPR>
static int run_write(WriteArgs& a, hipStream_t s, const char* who) {
  a.tokens = tokens_of((int64_t)a.p.H * LPR, 4);
  const int64_t x = std::max<int64_t>(((int64_t)a.T + a.tokens - 1) / a.tokens, 1);
  if (!countable(x)) return fail(PJX_ERR_INVALID, "pjx_write_pages: too many new tokens");
  launch_kernel<write_pages_kernel<E, QUANT, LPR>>(dim3((unsigned)x, (unsigned)std::min(a.B, 65535), 2), dim3(kPageThreads), 0, s, a);
  return check_launch(who);
}

template <typename E>
static int run_write(WriteArgs& a, bool quant, hipStream_t s, const char* who) {
  if (quant)
    return a.D <= 64    ? run_write<E, true, 8>(a, s, who)
           : a.D <= 128 ? run_write<E, true, 16>(a, s, who)
                        : run_write<E, true, 32>(a, s, who);
  const int lanes = a.D * fmt_size<E>() / 16;
  if constexpr (fmt_size<E>() == 4)
    if (lanes > 32) return run_write<E, false, 64>(a, s, who);
  return lanes <= 8    ? run_write<E, false, 8>(a, s, who)
         : lanes <= 16 ? run_write<E, false, 16>(a, s, who)
                       : run_write<E, false, 32>(a, s, who);
}

template <typename C, typename E>
static int run_read(ReadArgs& a, hipStream_t s, const char* who) {
  a.upr = a.D * fmt_size<E>() / 16;
  const int64_t per_token = (int64_t)a.p.H * a.upr;
  const bool stream = 2 * a.B * a.L * per_token * 16 >= kStreamRead;
  a.tokens = tokens_of(per_token, stream ? 8 : 4);
  a.by_token = fast_div(per_token);
  a.by_row = fast_div(a.upr);
  const int64_t x = (a.L + a.tokens - 1) / a.tokens;
  if (!countable(x)) return fail(PJX_ERR_INVALID, "pjx_read_pages: out_len is too long");
  const dim3 grid((unsigned)x, (unsigned)std::min(a.B, 65535), 2);
  if (stream) launch_kernel<read_pages_kernel<C, E, true>>(grid, dim3(kPageThreads), 0, s, a);
  else launch_kernel<read_pages_kernel<C, E, false>>(grid, dim3(kPageThreads), 0, s, a);
  return check_launch(who);
}

}  // namespace pjx

using namespace pjx;

extern "C" int pjx_write_pages(int dtype, int cache_dtype, const void* k, const void* v, const pjx_pages* cache,
                               const int32_t* kv_lengths, const int32_t* new_lengths, int32_t* lengths_out,
                               int64_t batch, int64_t len, int64_t kv_heads, int64_t head_dim,
                               const pjx_cache_strides* strides, void* stream) {
  clear_error();
  const char* who = "pjx_write_pages";
  WriteArgs a = {};
  const int rc = fill_pages(a.p, who, cache_dtype, cache, batch, kv_heads, head_dim);
  if (rc != PJX_OK) return rc;
  if (dtype != PJX_DTYPE_BF16 && dtype != PJX_DTYPE_F16 && dtype != PJX_DTYPE_F32)
    return fail(PJX_ERR_INVALID, "pjx_write_pages: dtype must be PJX_DTYPE_BF16, PJX_DTYPE_F16 or PJX_DTYPE_F32");
  const bool quant = cache_dtype == PJX_DTYPE_E4M3;
  if (!quant && cache_dtype != dtype) return fail(PJX_ERR_INVALID, "pjx_write_pages: the cache has another dtype");
  if (len < 0 || len > (1 << 30)) return fail(PJX_ERR_INVALID, "pjx_write_pages: sizes out of range");
  const int64_t size = dtype == PJX_DTYPE_F32 ? 4 : 2, row = kv_heads * head_dim, most = (int64_t)1 << 40;
  int64_t st[6] = {len * row, row, head_dim, len * row, row, head_dim};
  if (strides) {
    const int64_t given[6] = {strides->k_batch, strides->k_token, strides->k_head,
                              strides->v_batch, strides->v_token, strides->v_head};
    for (int i = 0; i < 6; ++i) {
      if (given[i] < 0 || given[i] > most) return fail(PJX_ERR_INVALID, "pjx_write_pages: strides out of range");
      if (given[i] * size % 16) return fail(PJX_ERR_INVALID, "pjx_write_pages: strides must be whole 16-byte chunks");
      st[i] = given[i];
    }
  }
  if (batch == 0) return PJX_OK;
  if (!lengths_out || (len > 0 && (!k || !v))) return fail(PJX_ERR_INVALID, "pjx_write_pages: null pointer");
  if (((uintptr_t)k | (uintptr_t)v) % 16) return fail(PJX_ERR_INVALID, "pjx_write_pages: k and v must start on 16 bytes");
  a.x[0] = (const char*)k; a.x[1] = (const char*)v;
  for (int i = 0; i < 2; ++i) {
    a.xb[i] = st[3 * i] * size; a.xt[i] = st[3 * i + 1] * size; a.xh[i] = st[3 * i + 2] * size;
  }
  a.lengths = kv_lengths; a.fresh = new_lengths; a.lengths_out = lengths_out;
  a.B = (int)batch; a.T = (int)len; a.D = (int)head_dim;
  a.by_h = fast_div(kv_heads);
  hipStream_t s = (hipStream_t)stream;
  return dtype == PJX_DTYPE_F32    ? run_write<F32Fmt>(a, quant, s, who)
         : dtype == PJX_DTYPE_BF16 ? run_write<Bf16Fmt>(a, quant, s, who)
                                   : run_write<F16Fmt>(a, quant, s, who);
}

extern "C" int pjx_read_pages(int dtype, int cache_dtype, const pjx_pages* cache, const int32_t* kv_lengths,
                              void* k_out, void* v_out, int64_t batch, int64_t out_len, int64_t kv_heads,
                              int64_t head_dim, void* stream) {
  clear_error();
  const char* who = "pjx_read_pages";
  ReadArgs a = {};
  const int rc = fill_pages(a.p, who, cache_dtype, cache, batch, kv_heads, head_dim);
  if (rc != PJX_OK) return rc;
  if (dtype != PJX_DTYPE_BF16 && dtype != PJX_DTYPE_F16 && dtype != PJX_DTYPE_F32)
    return fail(PJX_ERR_INVALID, "pjx_read_pages: dtype must be PJX_DTYPE_BF16, PJX_DTYPE_F16 or PJX_DTYPE_F32");
  const bool quant = cache_dtype == PJX_DTYPE_E4M3;
  if (!quant && cache_dtype != dtype) return fail(PJX_ERR_INVALID, "pjx_read_pages: the cache has another dtype");
  if (out_len < 0 || out_len > (1 << 30) || kv_heads * head_dim > (1 << 24))
    return fail(PJX_ERR_INVALID, "pjx_read_pages: sizes out of range");
  if (batch == 0 || out_len == 0) return PJX_OK;
  if (!k_out || !v_out) return fail(PJX_ERR_INVALID, "pjx_read_pages: null pointer");
  if (((uintptr_t)k_out | (uintptr_t)v_out) % 16)
    return fail(PJX_ERR_INVALID, "pjx_read_pages: k_out and v_out must start on 16 bytes");
  a.lengths = kv_lengths;
  a.y[0] = (char*)k_out; a.y[1] = (char*)v_out;
  a.B = (int)batch; a.D = (int)head_dim; a.L = out_len;
  hipStream_t s = (hipStream_t)stream;
  if (!quant)  // (a copy: the type's size alone matters)
    return dtype == PJX_DTYPE_F32 ? run_read<F32Fmt, F32Fmt>(a, s, who) : run_read<Bf16Fmt, Bf16Fmt>(a, s, who);
  return dtype == PJX_DTYPE_F32    ? run_read<E4m3Fmt, F32Fmt>(a, s, who)
         : dtype == PJX_DTYPE_BF16 ? run_read<E4m3Fmt, Bf16Fmt>(a, s, who)
                                   : run_read<E4m3Fmt, F16Fmt>(a, s, who);
}
