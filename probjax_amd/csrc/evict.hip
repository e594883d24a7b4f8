// Eviction from a KV cache for gfx950: every (sequence, KV head) keeps its first
// `sinks` and last `recent` keys and, of those between, the ones of the largest
// accumulated weight, in their order.
//
// Two kernels.  The selection runs one workgroup per (sequence, head), its weights
// in registers as order-preserving integers, and finds the threshold by counting
// digits of 11 bits in LDS, two or three passes; one more pass ranks the kept keys.
// It is bound by the latency of those steps and, of long caches, by the scalar unit
// that its 16 waves share (8 x 4096 weights 8.4 us, 128 x 8192 of them 11, 8 x 32768
// 31; read again in every pass, 2 x 40000: 46.  Bits counted two a round by ballots
// kept the scalar unit busy for 9 us more).  The gather reads and writes every kept K
// and V row once, 16 bytes a lane, bound by HBM (16 x 8192 keys of 8 heads of 128 cut
// to half their capacity, 490 MB: 97 us, 5.0 TB/s).
#include <stdio.h>

#include "pjx_common.h"
#include "pjx_internal.h"

namespace pjx {

struct EvictArgs {
  const uint32_t* weights;  // float bits
  const int32_t* lengths;
  uint32_t* weights_out;
  int32_t* lengths_out;
  int32_t* index;
  const char* x[2];  // k, v
  char* y[2];
  int64_t xb[2], xt[2], xh[2], yb[2], yt[2], yh[2];  // bytes
  int H, S, keep, out_len, sinks, recent, fill;
  int upr;         // units of a row (gather)
  uint32_t units;  // units of a sequence's kept rows
};

constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;

// Order-preserving integer of a weight: NaN above all, -0 as 0; never 0.
__device__ __forceinline__ uint32_t weight_key(uint32_t u) {
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (u == 0x80000000u) u = 0u;
  return u >> 31 ? ~u : u | 0x80000000u;
}

// R: weights of a thread's registers (the cache has at most R * kSelThreads); 0:
// read again in every pass.
constexpr int kTiles = 8;  // tiles of kSelThreads keys ranked, or loaded, together
constexpr int kDigit = 11, kBins = 1 << kDigit;
template <int R>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ __attribute__((aligned(8))) int bins[kBins];
  __shared__ int wave_sum[kSelWaves], found[3];
  __shared__ int rank_above[kTiles * kSelWaves], rank_at[kTiles * kSelWaves];
  __shared__ int total[2];
  static_assert(kSelWaves == 16 && kTiles * kSelWaves == 128, "two ranks per lane of a wave");
  static_assert(kBins == 2 * kSelThreads, "two bins per thread");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bh = blockIdx.x, b = bh / a.H;
  const int n = __builtin_amdgcn_readfirstlane(a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S);
  const int kept = min(n, a.keep);
  const uint32_t* w = a.weights + (size_t)bh * a.S;
  int32_t* index = a.index + (size_t)bh * a.keep;
  uint32_t* wout = a.weights_out + (size_t)bh * a.out_len;
  if (tid == 0 && bh % a.H == 0) a.lengths_out[b] = kept;
  for (int i = kept + tid; i < a.keep; i += kSelThreads) {
    index[i] = -1;
    if (a.fill) wout[i] = 0u;
  }
  if (n <= a.keep) {
    for (int i = tid; i < n; i += kSelThreads) {
      index[i] = i;
      wout[i] = w[i];
    }
    return;
  }
  // (loads without a condition: a branch around each would wait for it)
  auto weight_at = [&](int j) { return w[min(j, n - 1)]; };
  const int lo = a.sinks, hi = n - a.recent, need = a.keep - a.sinks - a.recent;
  auto key_of = [&](int j, uint32_t u) { return ((j >= lo) & (j < hi)) ? weight_key(u) : 0u; };  // 0: protected, or no key
  uint32_t raw[R > 0 ? R : kTiles];
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i) raw[i] = weight_at(tid + i * kSelThreads);
  }

  // T: the key of rank hi - lo - need from below among those between, kDigit bits a
  // pass: the keys that agree with T so far are counted by their next digit, and the
  // digit is the one in whose count the rank falls.
  uint32_t T = 0xffffffffu;
  int ties = 0;  // of the keys equal to T, so many are kept
  if (need > 0) {
    int2* own = (int2*)bins + tid;
    *own = {0, 0};
    __syncthreads();
    T = 0u;
    int skip = hi - lo - need;
#pragma unroll 1
    for (int shift = 32 - kDigit, known = 32;;) {
      auto look = [&](uint32_t u) {
        const bool in = (u != 0u) & (known == 32 || (u ^ T) >> (known & 31) == 0u);
        if (!in) return;
        // One atomic for all lanes of the first one's digit: weights often share one,
        // and atomics on one word take their turns.
        const int d = (int)(u >> shift) & (kBins - 1), d0 = __builtin_amdgcn_readfirstlane(d);
        const uint64_t same = __builtin_amdgcn_ballot_w64(d == d0);
        const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
        const int add = d != d0 ? 1 : before == 0 ? __popcll(same) : 0;
        if (add) atomicAdd(&bins[d], add);
      };
      if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) look(key_of(tid + i * kSelThreads, raw[i]));
      } else {
        for (int j0 = tid; j0 - tid < n; j0 += kTiles * kSelThreads) {
#pragma unroll
          for (int i = 0; i < kTiles; ++i) raw[i] = weight_at(j0 + i * kSelThreads);
#pragma unroll
          for (int i = 0; i < kTiles; ++i) look(key_of(j0 + i * kSelThreads, raw[i]));
        }
      }
      __syncthreads();
      const int2 c = *own;
      *own = {0, 0};
      const int sum = c.x + c.y, incl = wave_scan(sum);
      if (lane == 63) wave_sum[wave] = incl;
      __syncthreads();
      const int sums = row_scan(wave_sum[lane & 15]);
      const int first = (wave ? __builtin_amdgcn_readlane(sums, wave - 1) : 0) + incl - sum;
      if ((first <= skip) & (skip < first + sum)) {
        const bool y = skip >= first + c.x;
        found[0] = 2 * tid + y;
        found[1] = y ? first + c.x : first;  // keys of smaller digits
        found[2] = y ? c.y : c.x;
      }
      __syncthreads();
      const int digit = __builtin_amdgcn_readfirstlane(found[0]), count = __builtin_amdgcn_readfirstlane(found[2]);
      skip -= __builtin_amdgcn_readfirstlane(found[1]);
      T |= (uint32_t)digit << shift;
      if (skip == 0) {  // every key from T on is kept, whatever its further bits
        T -= 1;
        break;
      }
      if (shift == 0) {
        ties = count - skip;
        break;
      }
      known = shift;
      shift = max(shift - kDigit, 0);
    }
  }
  // Keys above T are kept, and of those at T the first `ties`.
  // Ranks, kTiles tiles at a time: every wave counts its kept and tied keys of each
  // tile, one wave sums them in the keys' order.
  int done_above = 0, done_at = 0;
  auto place = [&](int j0, const uint32_t* u) {
    uint64_t gm[kTiles], em[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const int j = j0 + i * kSelThreads + tid;
      const uint32_t x = key_of(j, u[i]);
      gm[i] = __builtin_amdgcn_ballot_w64((j < n) & ((x > T) | (x == 0u)));
      em[i] = __builtin_amdgcn_ballot_w64(x == T);
    }
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        rank_above[kSelWaves * i + wave] = __popcll(gm[i]);
        rank_at[kSelWaves * i + wave] = __popcll(em[i]);
      }
    }
    __syncthreads();
    if (wave < 2) {
      int* r = wave == 0 ? rank_above : rank_at;
      const int x = r[2 * lane], y = r[2 * lane + 1], end = wave_scan(x + y);
      r[2 * lane] = end - y - x;
      r[2 * lane + 1] = end - y;
      if (lane == 63) total[wave] = end;
    }
    __syncthreads();
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    int g0[kTiles], e0[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      g0[i] = done_above + rank_above[kSelWaves * i + wave] + __popcll(gm[i] & below);
      e0[i] = done_at + rank_at[kSelWaves * i + wave] + __popcll(em[i] & below);
    }
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      if ((gm[i] >> lane & 1) | ((em[i] >> lane & 1) & (e0[i] < ties))) {
        const int at = g0[i] + min(e0[i], ties);
        index[at] = j0 + i * kSelThreads + tid;
        wout[at] = u[i];
      }
    }
    done_above += total[0];
    done_at += total[1];
  };
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; i += kTiles)
      if (i * kSelThreads < n) {
        if (i > 0) __syncthreads();  // the last tiles' ranks have been read
        place(i * kSelThreads, raw + i);
      }
  } else {
    for (int j0 = 0; j0 < n; j0 += kTiles * kSelThreads) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) raw[i] = weight_at(j0 + i * kSelThreads + tid);
      __syncthreads();
      place(j0, raw);
    }
  }
}

// One unit (16 bytes, or an element where rows are no whole 16-byte chunks) of K
// and of V per thread and step.
constexpr int kGatherThreads = 256, kGatherUnits = 4;
template <typename U>
__global__ __launch_bounds__(kGatherThreads) void evict_gather_kernel(EvictArgs a) {
  const int b = blockIdx.y;
  const uint32_t base = blockIdx.x * (kGatherThreads * kGatherUnits) + threadIdx.x;
  U u[kGatherUnits][2];
  int64_t dst[kGatherUnits][2];
#pragma unroll
  for (int i = 0; i < kGatherUnits; ++i) {
    const uint32_t unit = base + i * kGatherThreads;
    dst[i][0] = -1;
    if (unit >= a.units) continue;
    const uint32_t row = unit / a.upr, c = unit - row * a.upr, slot = row / a.H, h = row - slot * a.H;
    const int j = a.index[((size_t)b * a.H + h) * a.keep + slot];
    if (j < 0 && !a.fill) continue;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      dst[i][w] = b * a.yb[w] + slot * a.yt[w] + h * a.yh[w] + (int64_t)c * sizeof(U);
      U z;
      __builtin_memset(&z, 0, sizeof(U));
      u[i][w] = z;
      if (j >= 0) u[i][w] = *(const U*)(a.x[w] + b * a.xb[w] + j * a.xt[w] + h * a.xh[w] + (int64_t)c * sizeof(U));
    }
  }
#pragma unroll
  for (int i = 0; i < kGatherUnits; ++i)
    if (dst[i][0] >= 0) {
#pragma unroll
      for (int w = 0; w < 2; ++w) *(U*)(a.y[w] + dst[i][w]) = u[i][w];
    }
}

}  // namespace pjx

using namespace pjx;

extern "C" int pjx_evict_keys(int64_t elem_size, const void* k, const void* v, const float* weights,
                              const int32_t* kv_lengths, void* k_out, void* v_out, float* weights_out,
                              int32_t* lengths_out, int32_t* index, int64_t batch, int64_t kv_len, int64_t kv_heads,
                              int64_t head_dim, int64_t out_len, int64_t keep, int64_t sinks, int64_t recent,
                              const pjx_cache_strides* strides, const pjx_cache_strides* out_strides, int fill,
                              void* stream) {
  clear_error();
  char buf[256];
  auto bad = [&](const char* what) {
    snprintf(buf, sizeof(buf), "pjx_evict_keys: %s", what);
    return fail(PJX_ERR_INVALID, buf);
  };
  if (elem_size != 2 && elem_size != 4) return bad("elem_size must be 2 or 4");
  if (batch < 0 || kv_len < 0 || kv_heads < 1 || head_dim < 1) return bad("bad sizes");
  if (keep < 0 || sinks < 0 || recent < 0 || sinks > keep || recent > keep - sinks)
    return bad("keep must be at least sinks + recent, all 0 or more");
  if (out_len < keep) return bad("out_len must be at least keep");
  const int64_t most = (int64_t)1 << 40;
  if (batch > 65535 || kv_len > (1 << 30) || out_len > (1 << 30) || kv_heads > (1 << 20) || head_dim > (1 << 16) ||
      batch * kv_heads > 0xffffffffLL / kSelThreads || keep * kv_heads > 0xff000000LL / head_dim)
    return bad("sizes out of range");
  if (batch == 0) return PJX_OK;
  if (!lengths_out || (keep > 0 && (!index || !k_out || !v_out || !weights_out)) ||
      (kv_len > 0 && (!weights || (keep > 0 && (!k || !v)))))
    return bad("null pointer");
  EvictArgs a = {};
  a.weights = (const uint32_t*)weights;
  a.lengths = kv_lengths;
  a.weights_out = (uint32_t*)weights_out;
  a.lengths_out = lengths_out;
  a.index = index;
  a.H = (int)kv_heads;
  a.S = (int)kv_len;
  a.keep = (int)keep;
  a.out_len = (int)out_len;
  a.sinks = (int)sinks;
  a.recent = (int)recent;
  a.fill = fill != 0;
  const int64_t row = kv_heads * head_dim;
  const pjx_cache_strides in_c = {kv_len * row, row, head_dim, kv_len * row, row, head_dim};
  const pjx_cache_strides out_c = {out_len * row, row, head_dim, out_len * row, row, head_dim};
  const pjx_cache_strides* st[2] = {strides ? strides : &in_c, out_strides ? out_strides : &out_c};
  bool chunks = head_dim * elem_size % 16 == 0;
  for (int i = 0; i < 2; ++i) {
    const int64_t s[6] = {st[i]->k_batch, st[i]->k_token, st[i]->k_head, st[i]->v_batch, st[i]->v_token, st[i]->v_head};
    for (int64_t x : s) {
      if (x < 0 || x > most) return bad("cache strides out of range");
      chunks = chunks && x * elem_size % 16 == 0;
    }
    int64_t* to[6] = {i ? &a.yb[0] : &a.xb[0], i ? &a.yt[0] : &a.xt[0], i ? &a.yh[0] : &a.xh[0],
                      i ? &a.yb[1] : &a.xb[1], i ? &a.yt[1] : &a.xt[1], i ? &a.yh[1] : &a.xh[1]};
    for (int j = 0; j < 6; ++j) *to[j] = s[j] * elem_size;
  }
  a.x[0] = (const char*)k; a.x[1] = (const char*)v;
  a.y[0] = (char*)k_out; a.y[1] = (char*)v_out;
  const uintptr_t all = (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_out | (uintptr_t)v_out;
  if (all % elem_size) return bad("pointers must be aligned to an element");
  chunks = chunks && all % 16 == 0;
  hipStream_t s = (hipStream_t)stream;
  const dim3 sel((unsigned)(batch * kv_heads));
  if (kv_len <= 8 * kSelThreads) launch_kernel<evict_select_kernel<8>>(sel, dim3(kSelThreads), 0, s, a);
  else if (kv_len <= 32 * kSelThreads) launch_kernel<evict_select_kernel<32>>(sel, dim3(kSelThreads), 0, s, a);
  else launch_kernel<evict_select_kernel<0>>(sel, dim3(kSelThreads), 0, s, a);
  int rc = check_launch("pjx_evict_keys");
  if (rc != PJX_OK || keep == 0) return rc;
  a.upr = (int)(chunks ? head_dim * elem_size / 16 : head_dim);
  a.units = (uint32_t)(keep * kv_heads * a.upr);
  const int64_t per = kGatherThreads * kGatherUnits;
  // (a launch counts its work-items along one axis in 32 bits: units < 2^32)
  const dim3 grid((unsigned)((a.units + per - 1) / per), (unsigned)batch);
  if (chunks) launch_kernel<evict_gather_kernel<u32x4>>(grid, dim3(kGatherThreads), 0, s, a);
  else if (elem_size == 4) launch_kernel<evict_gather_kernel<uint32_t>>(grid, dim3(kGatherThreads), 0, s, a);
  else launch_kernel<evict_gather_kernel<uint16_t>>(grid, dim3(kGatherThreads), 0, s, a);
  return check_launch("pjx_evict_keys");
}
