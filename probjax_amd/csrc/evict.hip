// Eviction from a KV cache for gfx950: every (sequence, KV head) keeps its first
// `sinks` and last `recent` keys and, of those between, the ones of the largest
// accumulated weight, in their order.
//
// Two kernels.  The selection runs one workgroup per (sequence, head), bound by
// the latency of its rounds: the weights stay in registers as order-preserving
// integers, the threshold is found two bits a round by counting (ballots, so the
// time does not depend on how the weights are spread, as that of a histogram in
// LDS does), and one more pass ranks the kept keys.  The gather reads and writes
// every kept K and V row once, 16 bytes a lane, bound by HBM.
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

// Sum over the 16 lanes of a row, in every lane of it.
__device__ __forceinline__ int row_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x128, 0xf, 0xf, false);  // row_ror:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x124, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x122, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x121, 0xf, 0xf, false);
  return x;
}

// Inclusive prefix sum over a wave.
__device__ __forceinline__ int wave_scan(int x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(x, d);
    x += lane >= d ? y : 0;
  }
  return x;
}

// R: keys of a thread's registers (the cache has at most R * kSelThreads); 0:
// read again in every round.
constexpr int kPlaceTiles = 8;  // tiles of kSelThreads keys ranked together
template <int R>
__global__ __launch_bounds__(kSelThreads) void evict_select_kernel(EvictArgs a) {
  __shared__ int count[2][3 * kSelWaves];
  __shared__ int rank_above[kPlaceTiles * kSelWaves], rank_at[kPlaceTiles * kSelWaves];
  __shared__ int total[2];
  static_assert(kSelWaves == 16 && kPlaceTiles * kSelWaves == 128, "two ranks per lane of a wave");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bh = blockIdx.x, b = bh / a.H;
  const int n = a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S;
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
  const int lo = a.sinks, hi = n - a.recent, need = a.keep - a.sinks - a.recent;
  auto key_at = [&](int j) { return j >= lo && j < hi ? weight_key(w[j]) : 0u; };  // 0: protected, or no key
  uint32_t key[R > 0 ? R : 1];
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; ++i) key[i] = key_at(tid + i * kSelThreads);
  }

  // T: the largest threshold that at least `need` keys reach, two bits a round;
  // above: how many reach the smallest one known to be too high.
  uint32_t T = 0;
  int above = 0;
  bool exact = false;  // exactly `need` keys reach T
  if (need == 0) {
    T = 0xffffffffu;
  } else {
    int round = 0;
    for (int bit = 30; bit >= 0 && !exact; bit -= 2, round ^= 1) {
      int c[3] = {0, 0, 0};
      auto look = [&](uint32_t u) {
#pragma unroll
        for (int j = 0; j < 3; ++j) c[j] += __popcll(__builtin_amdgcn_ballot_w64(u >= (T | (uint32_t)(j + 1) << bit)));
      };
      if constexpr (R > 0) {
#pragma unroll
        for (int i = 0; i < R; ++i) look(key[i]);
      } else {
        for (int j = tid; j < (n + kSelThreads - 1) / kSelThreads * kSelThreads; j += kSelThreads) look(key_at(j));
      }
      // (the counts are the same in every lane: the ballots' sums are scalars)
      if (lane < 3) count[round][16 * lane + wave] = lane == 0 ? c[0] : lane == 1 ? c[1] : c[2];
      __syncthreads();
      const int sums = row_sum(lane < 48 ? count[round][lane] : 0);
      int at = 0, reached = 0;
#pragma unroll
      for (int j = 2; j >= 0; --j) {  // the largest digit that enough keys reach
        const int sum = __builtin_amdgcn_readlane(sums, 16 * j);
        if (at == 0) {
          if (sum >= need) {
            at = j + 1;
            reached = sum;
          } else {
            above = sum;
          }
        }
      }
      T |= (uint32_t)at << bit;
      exact = at > 0 && reached == need;
    }
  }
  // Keys above T are kept, and of those at T the first `ties`.
  const int ties = need == 0 || exact ? 0 : need - above;
  if (exact) T -= 1;
  // Ranks, kPlaceTiles tiles at a time: every wave counts its kept and tied keys
  // of each tile, one wave sums them in the keys' order.
  int done_above = 0, done_at = 0;
  auto place = [&](int j0, const uint32_t* u) {
    uint64_t gm[kPlaceTiles], em[kPlaceTiles];
#pragma unroll
    for (int i = 0; i < kPlaceTiles; ++i) {
      const int j = j0 + i * kSelThreads + tid;
      gm[i] = __builtin_amdgcn_ballot_w64(j < n && (j < lo || j >= hi || u[i] > T));
      em[i] = __builtin_amdgcn_ballot_w64(j >= lo && j < hi && u[i] == T);
      if (lane == 0) {
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
#pragma unroll
    for (int i = 0; i < kPlaceTiles; ++i) {
      const int g0 = done_above + rank_above[kSelWaves * i + wave] + __popcll(gm[i] & below);
      const int e0 = done_at + rank_at[kSelWaves * i + wave] + __popcll(em[i] & below);
      if ((gm[i] >> lane & 1) || ((em[i] >> lane & 1) && e0 < ties)) {
        const int at = g0 + min(e0, ties), j = j0 + i * kSelThreads + tid;
        index[at] = j;
        wout[at] = w[j];
      }
    }
    done_above += total[0];
    done_at += total[1];
  };
  if constexpr (R > 0) {
#pragma unroll
    for (int i = 0; i < R; i += kPlaceTiles)
      if (i * kSelThreads < n) {
        if (i > 0) __syncthreads();  // the last tiles' ranks have been read
        place(i * kSelThreads, key + i);
      }
  } else {
    for (int j0 = 0; j0 < n; j0 += kPlaceTiles * kSelThreads) {
      uint32_t u[kPlaceTiles];
#pragma unroll
      for (int i = 0; i < kPlaceTiles; ++i) u[i] = key_at(j0 + i * kSelThreads + tid);
      __syncthreads();
      place(j0, u);
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
