// Rotary positions of one or several axes for gfx950.  The first
// R = sum(sections) features of a row form R/2 pairs, and pair p of a token at
// position x(axis(p)) turns by the angle x base^(-power(p)):
//   (a, b) -> (a cos - b sin, b cos + a sin);
// the gradient is the same kernel with the angles negated.
//
// Bound by HBM: every feature is read and written once.  Angles cost float64
// arithmetic (a position times a frequency loses the turn's fraction in float32
// from a few thousand on), so a workgroup forms the cosines and sines of its
// tokens once, in LDS, and all heads of q and k use them; a thread keeps its
// place within the rows, so it reads the table once per token.
#include <stdio.h>

#include "pjx_common.h"
#include "pjx_internal.h"

namespace pjx {

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 4;    // tokens of a workgroup at most
constexpr int kRotPairs = 128;   // rotated pairs of a row at most
constexpr int kRotAxes = 4;

struct RotaryArgs {
  const char* x[2];      // q, k (k may be absent)
  char* y[2];            // contiguous outputs
  int64_t sb[2], st[2], sh[2];  // bytes between sequences, tokens and heads of q and k
  int heads[2];          // heads of q, and of q and k together
  const void* pos;
  int64_t pos_b, pos_t;  // elements between sequences and tokens of the positions
  int pos_type;
  int axes, T, D;
  int64_t tokens;        // B * T
  int first_pair[kRotAxes + 1];  // pairs of axis a: first_pair[a] .. first_pair[a + 1]
  int interleaved, shared;
  double log2_base;
  float sign;
  int per_wg, heads_per_wg;
  int64_t block0;  // first block of a launch
};

__device__ __forceinline__ double rotary_position(const RotaryArgs& a, int64_t i) {
  switch (a.pos_type) {
    case PJX_POSITION_I32: return (double)((const int32_t*)a.pos)[i];
    case PJX_POSITION_I64: return (double)((const int64_t*)a.pos)[i];
    case PJX_POSITION_F32: return (double)((const float*)a.pos)[i];
    default: return ((const double*)a.pos)[i];
  }
}

// How a chunk's features find the other ones of their pairs.
constexpr int kInChunk = 0;   // interleaved: both in the chunk
constexpr int kChunk = 1;     // halves of whole chunks: in another chunk, at the same places
constexpr int kAnywhere = 2;  // one by one

// N elements of type T (uint16_t bits or float) as floats, and back.
template <typename E, int N>
struct RotChunk;
template <typename E>
struct RotChunk<E, 8> {
  typedef u32x4 raw;
  __device__ static void get(const char* p, float* v) {
    const u32x4 r = *(const u32x4*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = E::lo(r[i]);
      v[2 * i + 1] = E::hi(r[i]);
    }
  }
  __device__ static void put(char* p, const float* v) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = E::pack2(v[2 * i], v[2 * i + 1]);
    *(u32x4*)p = r;
  }
};
template <typename E>
struct RotChunk<E, 1> {
  __device__ static void get(const char* p, float* v) { v[0] = E::lo(*(const uint16_t*)p); }
  __device__ static void put(char* p, const float* v) { *(uint16_t*)p = E::bits(v[0]); }
};
struct F32Fmt {};
template <>
struct RotChunk<F32Fmt, 4> {
  __device__ static void get(const char* p, float* v) {
    const f32x4 r = *(const f32x4*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = r[i];
  }
  __device__ static void put(char* p, const float* v) { *(f32x4*)p = f32x4{v[0], v[1], v[2], v[3]}; }
};
template <>
struct RotChunk<F32Fmt, 1> {
  __device__ static void get(const char* p, float* v) { v[0] = *(const float*)p; }
  __device__ static void put(char* p, const float* v) { *(float*)p = v[0]; }
};

template <typename E, int N, int MODE>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotaryArgs a) {
  constexpr int SZ = std::is_same<E, F32Fmt>::value ? 4 : 2;
  __shared__ float2 turn[kRotTokens][kRotPairs];  // cos, sin
  const int tid = threadIdx.x;
  const int np = a.first_pair[a.axes];
  const int64_t n0 = (a.block0 + blockIdx.x) * a.per_wg;
  const int nt = (int)min((int64_t)a.per_wg, a.tokens - n0);

  for (int i = tid; i < nt * np; i += kRotThreads) {
    const int tok = i / np, p = i - tok * np;
    int axis = 0;
#pragma unroll
    for (int j = 1; j < kRotAxes; ++j)
      if (j < a.axes && p >= a.first_pair[j]) axis = j;
    const int lo = a.shared ? 0 : a.first_pair[axis], hi = a.shared ? np : a.first_pair[axis + 1];
    const int64_t n = n0 + tok, b = n / a.T, t = n - b * a.T;
    const double x = rotary_position(a, b * a.pos_b + t * a.pos_t + axis);
    // turns, less the whole ones
    const double f = exp2(-a.log2_base * (double)(p - lo) / (double)(hi - lo)) * 0.15915494309189535;
    const double r = x * f;
    float s, c;
    sincospif((float)(2.0 * (r - rint(r))), &s, &c);
    turn[tok][p] = make_float2(c, a.sign * s);
  }
  __syncthreads();

  // this thread's chunk within the rows, and the pair, side and partner of its features
  const int cpr = a.D / N, rows = kRotThreads / cpr;
  const int c = tid % cpr, r0 = tid / cpr;
  if (r0 >= rows) return;
  int pair[N], other[N];  // other: elements to the partner (kAnywhere: of each feature)
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const int d = N * c + e;
    pair[e] = -1;
    other[e] = 0;
    if (d >= 2 * np) continue;
    int lo = 0, hi = np;
    if (!a.shared) {
#pragma unroll
      for (int j = 0; j < kRotAxes; ++j)
        if (j < a.axes && d >= 2 * a.first_pair[j] && d < 2 * a.first_pair[j + 1]) {
          lo = a.first_pair[j];
          hi = a.first_pair[j + 1];
        }
    }
    const int in = d - 2 * lo, half = hi - lo;
    if (a.interleaved) {
      pair[e] = lo + in / 2;
      other[e] = in & 1 ? -1 : 1;
    } else {
      pair[e] = lo + (in < half ? in : in - half);
      other[e] = in < half ? half : -half;
    }
  }
  const int h_end = min((int)(blockIdx.y + 1) * a.heads_per_wg, a.heads[1]);
  for (int tok = 0; tok < nt; ++tok) {
    const int64_t n = n0 + tok, b = n / a.T, t = n - b * a.T;
    float co[N], si[N];  // out = x co + partner si
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float2 cs = pair[e] < 0 ? make_float2(1.f, 0.f) : turn[tok][pair[e]];
      co[e] = cs.x;
      si[e] = other[e] > 0 ? -cs.y : cs.y;
    }
#pragma unroll 2
    for (int h = blockIdx.y * a.heads_per_wg + r0; h < h_end; h += rows) {
      const int w = h >= a.heads[0], hh = w ? h - a.heads[0] : h, H = w ? a.heads[1] - a.heads[0] : a.heads[0];
      const char* row = a.x[w] + b * a.sb[w] + t * a.st[w] + hh * a.sh[w];
      const char* px = row + (int64_t)c * N * SZ;
      float v[N], o[N];
      RotChunk<E, N>::get(px, v);
      if constexpr (MODE == kInChunk) {
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = v[e ^ 1];
      } else if constexpr (MODE == kChunk) {
        RotChunk<E, N>::get(px + (int64_t)other[0] * SZ, o);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) RotChunk<E, 1>::get(px + (int64_t)(e + other[e]) * SZ, o + e);
      }
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float y = fmaf(v[e], co[e], o[e] * si[e]);
        v[e] = pair[e] < 0 ? v[e] : y;  // a feature that is not rotated passes whatever it holds
      }
      RotChunk<E, N>::put(a.y[w] + ((n * H + hh) * a.D + (int64_t)c * N) * SZ, v);
    }
  }
}

template <typename E, int N, int MODE>
static int launch_rotary(const RotaryArgs& a, int64_t blocks, hipStream_t s) {
  const int64_t most = 0xffffffffLL / kRotThreads;  // work-items of a launch: 32 bits
  const unsigned gy = (unsigned)((a.heads[1] + a.heads_per_wg - 1) / a.heads_per_wg);
  for (int64_t b = 0; b < blocks; b += most) {
    RotaryArgs args = a;
    args.block0 = b;
    launch_kernel<rotary_kernel<E, N, MODE>>(dim3((unsigned)std::min(most, blocks - b), gy), dim3(kRotThreads), 0, s,
                                             args);
  }
  return check_launch("pjx_rotary");
}

template <typename E, int N>
static int run_rotary(const RotaryArgs& a, int mode, bool chunks, int64_t blocks, hipStream_t s) {
  if (!chunks) return launch_rotary<E, 1, kAnywhere>(a, blocks, s);
  if (mode == kInChunk) return launch_rotary<E, N, kInChunk>(a, blocks, s);
  if (mode == kChunk) return launch_rotary<E, N, kChunk>(a, blocks, s);
  return launch_rotary<E, N, kAnywhere>(a, blocks, s);
}

}  // namespace pjx

using namespace pjx;

extern "C" int pjx_rotary(int dtype, const void* q, const void* k, void* q_out, void* k_out, const void* positions,
                          int position_type, int64_t position_batch_stride, int64_t position_token_stride,
                          int64_t batch, int64_t len, int64_t q_heads, int64_t k_heads, int64_t head_dim,
                          const pjx_cache_strides* strides, const int32_t* sections, int64_t axes, double base,
                          int interleaved, int shared_spectrum, int inverse, void* stream) {
  clear_error();
  char buf[256];
  auto bad = [&](const char* what) {
    snprintf(buf, sizeof(buf), "pjx_rotary: %s", what);
    return fail(PJX_ERR_INVALID, buf);
  };
  if (dtype != PJX_DTYPE_BF16 && dtype != PJX_DTYPE_F16 && dtype != PJX_DTYPE_F32)
    return bad("dtype must be PJX_DTYPE_BF16, PJX_DTYPE_F16 or PJX_DTYPE_F32");
  if (position_type < PJX_POSITION_I32 || position_type > PJX_POSITION_F64) return bad("position type");
  if (batch < 0 || len < 0 || q_heads < 0 || k_heads < 0 || head_dim < 1 || head_dim > 256 ||
      q_heads + k_heads > (1 << 20) || batch > (1 << 30) || len > (1 << 30) || batch * len > ((int64_t)1 << 40))
    return bad("sizes out of range (head_dim at most 256)");
  if (axes < 1 || axes > kRotAxes || !sections) return bad("1 to 4 axes");
  if (!(base > 0.0) || base > 1e300) return bad("base must be a positive number");
  if (position_batch_stride < 0 || position_token_stride < 0) return bad("position strides");
  RotaryArgs a = {};
  int width = 0;
  for (int i = 0; i < axes; ++i) {
    if (sections[i] < 0 || sections[i] % 2 || sections[i] > head_dim) return bad("sections must be even, 0 or more");
    a.first_pair[i] = width / 2;
    width += sections[i];
  }
  a.first_pair[axes] = width / 2;
  if (width > head_dim) return bad("sections exceed head_dim");
  const int64_t rows = q_heads + k_heads;
  if (batch * len * rows == 0) return PJX_OK;
  if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || !positions) return bad("null pointer");
  const bool f32 = dtype == PJX_DTYPE_F32;
  const int sz = f32 ? 4 : 2, n = 16 / sz;
  const int64_t d = head_dim;
  const int64_t el[2][3] = {{strides ? strides->k_batch : len * q_heads * d, strides ? strides->k_token : q_heads * d,
                             strides ? strides->k_head : d},
                            {strides ? strides->v_batch : len * k_heads * d, strides ? strides->v_token : k_heads * d,
                             strides ? strides->v_head : d}};
  bool chunks = d % n == 0;
  const void* x[2] = {q, k};
  void* y[2] = {q_out, k_out};
  const int64_t heads[2] = {q_heads, k_heads};
  for (int i = 0; i < 2; ++i) {
    if (!heads[i]) continue;
    for (int64_t s : el[i]) {
      if (s < 0 || s > ((int64_t)1 << 40)) return bad("strides out of range");
      chunks = chunks && s % n == 0;
    }
    if ((uintptr_t)x[i] % sz || (uintptr_t)y[i] % sz) return bad("pointers must be aligned to an element");
    chunks = chunks && (uintptr_t)x[i] % 16 == 0 && (uintptr_t)y[i] % 16 == 0;
    a.x[i] = (const char*)x[i];
    a.y[i] = (char*)y[i];
    a.sb[i] = el[i][0] * sz;
    a.st[i] = el[i][1] * sz;
    a.sh[i] = el[i][2] * sz;
  }
  a.heads[0] = (int)q_heads;
  a.heads[1] = (int)rows;
  a.pos = positions;
  a.pos_type = position_type;
  a.pos_b = position_batch_stride;
  a.pos_t = position_token_stride;
  a.axes = (int)axes;
  a.T = (int)len;
  a.D = (int)d;
  a.tokens = batch * len;
  a.interleaved = interleaved != 0;
  a.shared = shared_spectrum != 0;
  a.log2_base = log2(base);
  a.sign = inverse ? -1.f : 1.f;
  int mode = kInChunk;
  if (!a.interleaved) {
    // halves of whole chunks that start on one
    bool whole = true;
    if (a.shared) whole = width / 2 % n == 0;
    else
      for (int i = 0; i < axes; ++i) whole = whole && sections[i] / 2 % n == 0;
    mode = whole ? kChunk : kAnywhere;
  }
  // Few tokens: a workgroup takes one, and their heads spread over several.
  const int64_t want = 1024;
  a.per_wg = (int)std::clamp<int64_t>(a.tokens / want, 1, kRotTokens);
  const int64_t blocks = (a.tokens + a.per_wg - 1) / a.per_wg;
  const int rows_per_pass = std::max<int>(1, kRotThreads / (int)(chunks ? d / n : d));
  const int64_t most_y = (rows + rows_per_pass - 1) / rows_per_pass;
  const int64_t gy = std::clamp<int64_t>(want / blocks, 1, most_y);
  a.heads_per_wg = (int)((rows + gy - 1) / gy);
  hipStream_t s = (hipStream_t)stream;
  if (f32) return run_rotary<F32Fmt, 4>(a, mode, chunks, blocks, s);
  return dtype == PJX_DTYPE_F16 ? run_rotary<F16Fmt, 8>(a, mode, chunks, blocks, s)
                                : run_rotary<Bf16Fmt, 8>(a, mode, chunks, blocks, s);
}
