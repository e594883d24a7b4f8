// Rotary positions of one or several axes for gfx950.  The first
// R = sum(sections) features of a row form R/2 pairs, and pair p of a token at
// position x(axis(p)) turns by the angle x base^(-power(p)):
//   (a, b) -> (a cos - b sin, b cos + a sin);
// the gradient is the same kernel with the angles negated.
//
// Bound by HBM: every feature is read and written once.  Angles cost float64
// arithmetic (a position times a frequency loses the turn's fraction in float32
// from a few thousand on), so a workgroup forms the cosines and sines of its
// tokens once, in LDS, and all heads of q and k use them.  A thread keeps its place
// within the rows and takes four of them at a time, their loads issued before the
// first store.  The products and the sum are float32, rounded to the type once.  bf16,
// 12288 tokens of 16 + 16 heads of 128 (201 MB): 45 us interleaved, 4.5 TB/s; halves,
// 2 x 4096 tokens of 16 + 4 heads (84 MB): 21.6 us, 3.9 TB/s; one row a thread at a
// time took 51 and 30.
#include <stdio.h>

#include "pjx_common.h"
#include "pjx_internal.h"

namespace pjx {

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 16;   // tokens of a workgroup at most
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
  int tokens;            // B * T
  int first_pair[kRotAxes + 1];  // pairs of axis a: first_pair[a] .. first_pair[a + 1]
  int interleaved, shared;
  double rate[kRotAxes];  // log2 of the frequency's step from pair to pair
  float sign;
  int per_wg, heads_per_wg;
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

// A chunk of N elements of format E in memory and as floats.
struct F32Fmt {};
template <typename E, int N>
struct RotChunk;
template <typename E>
struct RotChunk<E, 8> {
  typedef u32x4 raw;
  __device__ static void get(const raw& r, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = E::lo(r[i]);
      v[2 * i + 1] = E::hi(r[i]);
    }
  }
  __device__ static raw put(const float* v) {
    return raw{E::pack2(v[0], v[1]), E::pack2(v[2], v[3]), E::pack2(v[4], v[5]), E::pack2(v[6], v[7])};
  }
};
template <typename E>
struct RotChunk<E, 1> {
  typedef uint16_t raw;
  __device__ static void get(raw r, float* v) { v[0] = E::lo(r); }
  __device__ static raw put(const float* v) { return E::bits(v[0]); }
};
template <>
struct RotChunk<F32Fmt, 4> {
  typedef f32x4 raw;
  __device__ static void get(const raw& r, float* v) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = r[i];
  }
  __device__ static raw put(const float* v) { return raw{v[0], v[1], v[2], v[3]}; }
};
template <>
struct RotChunk<F32Fmt, 1> {
  typedef float raw;
  __device__ static void get(raw r, float* v) { v[0] = r; }
  __device__ static raw put(const float* v) { return v[0]; }
};

template <typename E, int N, int MODE>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotaryArgs a) {
  typedef RotChunk<E, N> C;
  typedef typename C::raw Raw;
  typedef RotChunk<E, 1> One;
  constexpr int SZ = std::is_same<E, F32Fmt>::value ? 4 : 2;
  constexpr int CH = MODE == kChunk ? 2 : 1;          // chunks of a thread's unit
  constexpr int ROWS = MODE == kChunk ? 2 : 4;        // rows of a thread at a time
  __shared__ float2 turn[kRotTokens * kRotPairs];     // cos, sin of pair p of token t at t * pairs + p
  const int tid = threadIdx.x;
  const int np = a.first_pair[a.axes];
  const int n0 = blockIdx.x * a.per_wg, nt = min(a.per_wg, a.tokens - n0);

  for (int i = tid; i < nt * np; i += kRotThreads) {
    const int tok = i / np, p = i - tok * np;
    int axis = 0;
#pragma unroll
    for (int j = 1; j < kRotAxes; ++j)
      if (j < a.axes && p >= a.first_pair[j]) axis = j;
    const int n = n0 + tok, b = n / a.T, t = n - b * a.T;
    const double x = rotary_position(a, b * a.pos_b + t * a.pos_t + axis);
    double rate = a.rate[0];
#pragma unroll
    for (int j = 1; j < kRotAxes; ++j) rate = axis == j ? a.rate[j] : rate;
    int lo = a.first_pair[0];
#pragma unroll
    for (int j = 1; j < kRotAxes; ++j) lo = axis == j && !a.shared ? a.first_pair[j] : lo;
    // turns, less the whole ones
    const double r = x * (exp2(rate * (double)(p - lo)) * 0.15915494309189535);
    float s, c;
    sincospif((float)(2.0 * (r - rint(r))), &s, &c);
    turn[i] = make_float2(c, a.sign * s);
  }

  // This thread's unit of a row: its first feature (kChunk: of the first half, the
  // second `apart` features on), its first pair, how many of its features turn.
  const int units = MODE == kChunk ? np / N + (a.D - 2 * np) / N : a.D / N;
  const int per_pass = kRotThreads / units;
  const int u = tid % units, r0 = tid / units;
  int d0 = N * u, apart = 0, pair0 = N * u / 2, turns = min(max(2 * np - N * u, 0), N);
  if constexpr (MODE == kChunk) {
    int lo = 0, hi = np;
    if (!a.shared) {
#pragma unroll
      for (int j = 0; j < kRotAxes; ++j)
        if (j < a.axes && N * u >= a.first_pair[j] && N * u < a.first_pair[j + 1]) {
          lo = a.first_pair[j];
          hi = a.first_pair[j + 1];
        }
    }
    pair0 = N * u;
    turns = N * u < np ? N : 0;
    d0 = turns ? lo + N * u : N * u + np;
    apart = hi - lo;
  }
  int pair[MODE == kAnywhere ? N : 1], other[MODE == kAnywhere ? N : 1];  // of each feature, elements to its partner
  if constexpr (MODE == kAnywhere) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int d = d0 + e;
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
      const bool first = a.interleaved ? !(in & 1) : in < half;
      pair[e] = d < 2 * np ? lo + (a.interleaved ? in / 2 : first ? in : in - half) : 0;
      other[e] = d < 2 * np ? (a.interleaved ? 1 : half) * (first ? 1 : -1) : 0;
    }
  }
  __syncthreads();
  if (r0 >= per_pass) return;

  const int h0 = blockIdx.y * a.heads_per_wg, nh = min(a.heads_per_wg, a.heads[1] - h0);
  const int last = nt * nh;
  for (int i0 = r0; i0 < last; i0 += ROWS * per_pass) {
    Raw v[ROWS][CH];
    char* to[ROWS];
    int tok[ROWS];
    float o[ROWS][MODE == kAnywhere ? N : 1];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int row = i0 + i * per_pass;
      if (row >= last) break;
      tok[i] = row / nh;
      const int h = h0 + row - tok[i] * nh, n = n0 + tok[i], b = n / a.T, t = n - b * a.T;
      const int w = h >= a.heads[0], hh = w ? h - a.heads[0] : h, H = w ? a.heads[1] - a.heads[0] : a.heads[0];
      const char* px = a.x[w] + b * a.sb[w] + t * a.st[w] + hh * a.sh[w] + d0 * SZ;
      to[i] = a.y[w] + (((int64_t)n * H + hh) * a.D + d0) * SZ;
      v[i][0] = *(const Raw*)px;
      if constexpr (MODE == kChunk)
        if (turns) v[i][1] = *(const Raw*)(px + apart * SZ);
      if constexpr (MODE == kAnywhere)
#pragma unroll
        for (int e = 0; e < N; ++e) One::get(*(const typename One::raw*)(px + (e + other[e]) * SZ), o[i] + e);
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (i0 + i * per_pass >= last) break;
      const float2* cs = turn + tok[i] * np;
      if (turns == 0) {  // features that are not rotated pass whatever they hold
        *(Raw*)to[i] = v[i][0];
        continue;
      }
      float x[N], y[N];
      C::get(v[i][0], x);
      if constexpr (MODE == kInChunk) {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const float2 k = cs[pair0 + min(e, turns - 2) / 2];
          y[e] = e < turns ? fmaf(x[e], k.x, -x[e + 1] * k.y) : x[e];
          y[e + 1] = e < turns ? fmaf(x[e + 1], k.x, x[e] * k.y) : x[e + 1];
        }
      } else if constexpr (MODE == kChunk) {
        float z[N], q[N];
        C::get(v[i][1], z);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float2 k = cs[pair0 + e];
          y[e] = fmaf(x[e], k.x, -z[e] * k.y);
          q[e] = fmaf(z[e], k.x, x[e] * k.y);
        }
        *(Raw*)(to[i] + apart * SZ) = C::put(q);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float2 k = cs[pair[e]];
          const float s = other[e] > 0 ? -k.y : k.y;
          y[e] = e < turns ? fmaf(x[e], k.x, o[i][e] * s) : x[e];
        }
      }
      *(Raw*)to[i] = C::put(y);
    }
  }
}

template <typename E, int N, int MODE>
static int launch_rotary(RotaryArgs& a, hipStream_t s) {
  // Tokens of a workgroup: enough for a round or more of its threads' rows; where
  // that leaves few workgroups, fewer, and the heads of one spread over several.
  const int64_t np = a.first_pair[a.axes], rows = a.heads[1];
  const int64_t units = MODE == kChunk ? np / N + (a.D - 2 * np) / N : a.D / N, per_pass = kRotThreads / units;
  const int64_t want = 1024, full = (8 / (MODE == kChunk ? 2 : 1) * per_pass + rows - 1) / rows;
  a.per_wg = (int)std::clamp<int64_t>(std::min<int64_t>(full, a.tokens / want), 1, kRotTokens);
  const int64_t blocks = (a.tokens + a.per_wg - 1) / a.per_wg;
  const int64_t gy = std::clamp<int64_t>(want / blocks, 1, (rows + per_pass - 1) / per_pass);
  a.heads_per_wg = (int)((rows + gy - 1) / gy);
  if (blocks > 0xffffffffLL / kRotThreads) return fail(PJX_ERR_INVALID, "pjx_rotary: too many tokens");
  const dim3 grid((unsigned)blocks, (unsigned)((rows + a.heads_per_wg - 1) / a.heads_per_wg));
  launch_kernel<rotary_kernel<E, N, MODE>>(grid, dim3(kRotThreads), 0, s, a);
  return check_launch("pjx_rotary");
}

template <typename E, int N>
static int run_rotary(RotaryArgs& a, int mode, bool chunks, hipStream_t s) {
  if (!chunks) return launch_rotary<E, 1, kAnywhere>(a, s);
  if (mode == kInChunk) return launch_rotary<E, N, kInChunk>(a, s);
  if (mode == kChunk) return launch_rotary<E, N, kChunk>(a, s);
  return launch_rotary<E, N, kAnywhere>(a, s);
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
      q_heads + k_heads > (1 << 20) || batch > (1 << 30) || len > (1 << 30) || batch > 0x7fffffffLL / std::max<int64_t>(len, 1))
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
  a.tokens = (int)(batch * len);
  a.interleaved = interleaved != 0;
  a.shared = shared_spectrum != 0;
  for (int i = 0; i < axes; ++i) {
    const int pairs = a.shared ? width / 2 : sections[i] / 2;
    a.rate[i] = pairs > 0 ? -log2(base) / pairs : 0.0;
  }
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
  hipStream_t s = (hipStream_t)stream;
  if (f32) return run_rotary<F32Fmt, 4>(a, mode, chunks, s);
  return dtype == PJX_DTYPE_F16 ? run_rotary<F16Fmt, 8>(a, mode, chunks, s)
                                : run_rotary<Bf16Fmt, 8>(a, mode, chunks, s);
}
