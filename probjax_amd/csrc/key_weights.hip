// The softmax weight that every key of a cache was given, for gfx950:
//   w'[b, g, j] = w[b, g, j] + sum over the rows t and heads h of group g of
//                 exp(s_htj - lse_ht),
// what eviction from a KV cache goes by (evict.hip).
//
// Decode steps (few rows): the split-KV decode (decode_common.h) also keeps its
// scores, 4 bytes a row and key beside the 2 (D + D) bytes of a 16-bit key, and
// a second kernel sums their exponentials once the rows' statistics are known.
// Forming the scores again instead would read K, half of the cache, again.  bf16, 8 KV
// heads of 128, 4 rows each: 32 sequences of 512 .. 8192 keys (588 MB) 118 us, bound by
// HBM (the decode without scores 107), and 11 us for the second kernel; one of 4096
// keys 8 and 4.7 us, bound by latency.
//
// Prompts (many rows): the scores are too many to keep.  They are formed again
// on the matrix units, keys as MFMA rows, so a lane's accumulators are sums of
// its own 16 keys and nothing is exchanged until the end.  bf16, 4096 causal rows of
// 16 heads over 4 KV heads of 128: 57 to 59 us, 590 to 600 TFLOP/s; the sum over the
// splits 4.6 us.  No unit bounds it alone: while a CU is busy its matrix units work 41%
// of the cycles and its VALUs 55% (a third of that exponentials, one for every 256
// operations), two waves a SIMD, which leave gaps at each tile's barrier; and the CUs
// are busy 77% of the time, the causal halves of the workgroups being uneven.
//
// Scores, their exponentials and every sum are float32, in a fixed order.
#include <stdio.h>

#include "decode_common.h"
#include "flash_common.h"

namespace pjx {

template <typename E, int D, int NRB, bool STREAM, bool ROWS>
__global__ __launch_bounds__(256, (decode_occupancy<D, D, NRB>())) void scored_decode_kernel(DecodeArgs a) {
  gqa_decode<E, D, D, NRB, STREAM, ROWS, kScores>(a);
}

template <int D, int NRB>
__global__ __launch_bounds__(256, 1) void scored_decode_f32_kernel(DecodeArgs a) {
  gqa_decode_f32<D, D, NRB, kScores>(a);
}

constexpr int kWeightThreads = 128;  // the merge's, which shares the launch
constexpr int kWeightKeys = 4 * kWeightThreads;
constexpr int kMaxScoredRows = 64;
constexpr int kRowsAhead = 4;
static_assert(kWeightThreads == kMergeThreads && kMaxScoredRows <= kWeightThreads, "one launch");

// After the chunk kernel: the first merge_blocks workgroups merge the outputs,
// every further one forms the weights of 512 keys, 4 consecutive ones a thread.
// Each of these finds the statistics of its rows itself, from the chunks'.
__global__ __launch_bounds__(kWeightThreads) void scored_merge_kernel(DecodeArgs a, const float* w_in, float* w_out,
                                                                     int merge_blocks, int key_blocks) {
  if ((int)blockIdx.x < merge_blocks) {
    merge_chunks(a, (long)blockIdx.x * kWeightThreads + threadIdx.x);
    return;
  }
  __shared__ float2 stat[kMaxScoredRows];  // running max (log2 units), 1 / sum
  const int block = blockIdx.x - merge_blocks, bg = block / key_blocks;
  const int b = bg / a.G, tid = threadIdx.x;
  const int L = seq_len(a, b), n = (L + a.chunk - 1) / a.chunk;
  const int j0 = block % key_blocks * kWeightKeys + 4 * tid;
  // The weights so far and, of few rows, the scores, on their way while the statistics
  // are found (4 rows, 32 sequences of 512 .. 8192 keys: 131.8 -> 129.7 us for the step).
  const float* s = a.scores + (size_t)bg * a.rows * a.score_ld + j0;
  f32x4 first[kRowsAhead] = {};
  const bool ahead = a.rows <= kRowsAhead;
  if (ahead && j0 < L)
#pragma unroll
    for (int r = 0; r < kRowsAhead; ++r) first[r] = *(const f32x4*)(s + (size_t)min(r, a.rows - 1) * a.score_ld);
  const size_t at = (size_t)bg * a.Lk + j0;
  float w[4] = {};
  if (w_in)
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = w_in[(size_t)bg * a.Lk + min(j0 + e, a.Lk - 1)];
  // each row's chunks over the lanes it gets: a power of two of them, in one wave
  int per = 64;
  while (per * a.rows > kWeightThreads) per /= 2;
  const int row = tid / per, l0 = tid % per;
  float M = kMaxInit, sum = 0.f;
  if (row < a.rows) {
    const float2* ml = (const float2*)a.ws_ml + (size_t)bg * a.nch * a.rows + row;
    for (int c = l0; c < n; c += per) {
      const float2 x = ml[(size_t)c * a.rows];
      const float m_new = fmaxf(M, x.x);
      sum = fmaf(sum, fast_exp2(M - m_new), x.y * fast_exp2(x.x - m_new));
      M = m_new;
    }
  }
  for (int d = per / 2; d > 0; d /= 2) {
    const float m2 = __shfl_xor(M, d), s2 = __shfl_xor(sum, d), m_new = fmaxf(M, m2);
    sum = sum * fast_exp2(M - m_new) + s2 * fast_exp2(m2 - m_new);
    M = m_new;
  }
  if (row < a.rows && l0 == 0) stat[row] = make_float2(M, 1.f / sum);
  __syncthreads();
  if (j0 >= a.Lk) return;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](const f32x4& x, const float2 st) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(fast_exp2(x[e] - st.x), st.y, acc[e]);
  };
  if (ahead) {
#pragma unroll
    for (int r = 0; r < kRowsAhead; ++r)
      if (r < a.rows) add(first[r], stat[r]);
  } else if (j0 < L) {
#pragma unroll 4
    for (int r = 0; r < a.rows; ++r) add(*(const f32x4*)(s + (size_t)r * a.score_ld), stat[r]);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (j0 + e < a.Lk) w_out[at + e] = w[e] + (j0 + e < L ? acc[e] : 0.f);
}

template <auto K>
static int run_scored(DecodeArgs& a, const float* w_in, float* w_out, void* ws, size_t ws_bytes, hipStream_t s) {
  const char* who = "pjx_weighted_decode";
  const int rc = run_chunks<K>(a, ws, ws_bytes, s, who);
  if (rc != PJX_OK) return rc;
  const int64_t merge = ((int64_t)a.B * a.G * a.rows * (a.orow / 4) + kWeightThreads - 1) / kWeightThreads;
  const int64_t keys = (a.Lk + kWeightKeys - 1) / kWeightKeys, blocks = merge + keys * a.B * a.G;
  if (blocks > 0xffffffffLL / kWeightThreads) return fail(PJX_ERR_INVALID, "pjx_weighted_decode: sizes out of range");
  launch_kernel<scored_merge_kernel>(dim3((unsigned)blocks), dim3(kWeightThreads), 0, s, a, w_in, w_out, (int)merge,
                                     (int)keys);
  return check_launch(who);
}

// Caches past decode_streams_kv's threshold are read with non-temporal loads, as
// the plain decode reads them (up to 32 rows at head dims up to 128).
template <typename E, int D, bool ROWS>
static int run_scored_rows(DecodeArgs& a, int nrb, const float* wi, float* wo, void* ws, size_t n, hipStream_t s) {
  if constexpr (!ROWS && D <= 128) {
    if (nrb <= 2 && decode_streams_kv((int64_t)a.B * a.Lk * a.G * 2 * D * 2, kStreamBytes))
      return nrb == 1 ? run_scored<scored_decode_kernel<E, D, 1, true, false>>(a, wi, wo, ws, n, s)
                      : run_scored<scored_decode_kernel<E, D, 2, true, false>>(a, wi, wo, ws, n, s);
  }
  if (nrb == 1) return run_scored<scored_decode_kernel<E, D, 1, false, ROWS>>(a, wi, wo, ws, n, s);
  if (nrb == 2) return run_scored<scored_decode_kernel<E, D, 2, false, ROWS>>(a, wi, wo, ws, n, s);
  if constexpr (D <= 128) return run_scored<scored_decode_kernel<E, D, 4, false, ROWS>>(a, wi, wo, ws, n, s);
  return fail(PJX_ERR_INVALID, "pjx_weighted_decode: row blocks");
}

template <typename E>
static int run_scored_16(DecodeArgs& a, int d, int nrb, const float* wi, float* wo, void* ws, size_t n, hipStream_t s) {
  const bool rows = a.orow != d;
  if (d == 64)
    return rows ? run_scored_rows<E, 64, true>(a, nrb, wi, wo, ws, n, s)
                : run_scored_rows<E, 64, false>(a, nrb, wi, wo, ws, n, s);
  if (d == 128)
    return rows ? run_scored_rows<E, 128, true>(a, nrb, wi, wo, ws, n, s)
                : run_scored_rows<E, 128, false>(a, nrb, wi, wo, ws, n, s);
  return run_scored_rows<E, 256, false>(a, nrb, wi, wo, ws, n, s);
}

template <int D>
static int run_scored_f32(DecodeArgs& a, int nrb, const float* wi, float* wo, void* ws, size_t n, hipStream_t s) {
  return nrb == 1 ? run_scored<scored_decode_f32_kernel<D, 1>>(a, wi, wo, ws, n, s)
                  : run_scored<scored_decode_f32_kernel<D, 2>>(a, wi, wo, ws, n, s);
}

// The automatic chunk: the decode's, up to 1024 keys.  MI355X, us, 1024 / 2048 keys,
// 8 KV heads of 128, 4 rows each: 32 sequences of 512 .. 8192 keys 130 / 137, 8 of up to
// 32768 130 / 140, 32 full ones of 8192 221 / 218.
static int64_t scored_chunk(int64_t batch, int64_t groups, int64_t kv_len, int64_t chunk) {
  return chunk ? chunk : std::min<int64_t>(auto_chunk(batch, groups, kv_len, kGqaItems), 1024);
}

// Workspace of a weighted decode: the decode's partials, then the scores.
static size_t partial_bytes(int64_t batch, int64_t groups, int64_t rows, int64_t kv_len, int64_t v_dim, int64_t chunk) {
  return (ws_size(batch, groups, rows, kv_len, v_dim, chunk) + 255) & ~(size_t)255;
}
static int64_t score_stride(int64_t kv_len) { return (kv_len + 3) & ~(int64_t)3; }

// ---------------------------------------------------------------------------
// Prompts
// ---------------------------------------------------------------------------
struct KeyWeightArgs {
  const void* q;
  const void* k;
  const float* lse;
  const int32_t* lengths;
  float* part;  // [splits][B * G][Lk]
  int B, Lq, Lk, Hq, G, rdim;
  int causal, shift;
  int q_step;   // query rows of a split
  int splits;   // splits of the query rows (each per head)
  float cx;
};

// Keys of a wave, in blocks of 32 (their fragments stay in registers): a query
// fragment read from LDS serves all of them.  With one block, the four waves'
// reads of a query tile take as long as their products.
constexpr int key_blocks(int head_dim) { return head_dim <= 128 ? 2 : 1; }

// What a workgroup works on: keys k_first .. of one (batch, KV head), against the
// query rows [q_lo, q_hi) of one split of one head of its group.
struct KeyWork {
  int b, g, h, hs, L, q_lo, q_hi;
};
// Workgroup x works on key block x / (rows of the grid); of the rest, heads vary
// slower than splits, and the split is turned by the key block and the head: under
// a causal mask early splits and late key blocks have little to do, and workgroup
// x runs on XCD x % 8, so any fixed order gives some XCDs the heavy ones (key
// block fastest: 100 us for 70 on the prompt below).
__device__ __forceinline__ KeyWork key_work(const KeyWeightArgs& a, int keys, int& k_first) {
  KeyWork u;
  const int per = a.Hq / a.G, units = a.B * a.Hq * a.splits;
  const int block = blockIdx.x / units, y = blockIdx.x % units, hb = y / a.splits;
  const int split = (y + hb + block) % a.splits;
  k_first = block * keys;
  u.b = hb / a.Hq;
  u.h = hb % a.Hq;
  u.g = u.h / per;
  u.hs = u.h % per * a.splits + split;
  // (a scalar: loaded as a vector, everything up to the loop's count became one)
  u.L = a.lengths ? min(a.Lk, max(__builtin_amdgcn_readfirstlane(a.lengths[u.b]), 0)) : a.Lk;
  u.q_lo = split * a.q_step;
  u.q_hi = min(u.q_lo + a.q_step, a.Lq);
  // (rows before it see none of the keys)
  if (a.causal) u.q_lo = max(u.q_lo, max(k_first - a.shift, 0) / 32 * 32);
  if (k_first >= u.L) u.q_hi = u.q_lo;
  return u;
}

template <int N>
__device__ __forceinline__ void halve(float* x, int d) {
  const bool up = (threadIdx.x & d) != 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float keep = x[i], give = x[i + N];
    asm volatile("" : "+v"(keep), "+v"(give));  // (two selects; merged over the registers they became hundreds)
    const float k = up ? give : keep, g = up ? keep : give;
    x[i] = k + __shfl_xor(g, d);
  }
}

// Writes the sums over the 32 queries of a half wave of one block of 32 keys.
// Each exchange halves the registers: a lane keeps the half that its bit names and
// adds its partner's, so 16 exchanges do for 16 registers; lane c ends with
// register bit-reverse(c % 16).
__device__ __forceinline__ void put_weights(const KeyWeightArgs& a, const KeyWork& u, const f32x16& sums, int k0) {
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  float* part = a.part + ((size_t)u.hs * a.B * a.G + u.b * a.G + u.g) * a.Lk;
  float x[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) x[r] = sums[r];
  if (u.q_lo < u.q_hi) {
    halve<8>(x, 1);
    halve<4>(x, 2);
    halve<2>(x, 4);
    halve<1>(x, 8);
    x[0] += __shfl_xor(x[0], 16);
  }
  const int r = (col & 1) << 3 | (col & 2) << 1 | (col & 4) >> 1 | (col & 8) >> 3;
  const int key = k0 + 8 * (r >> 2) + 4 * half + (r & 3);
  if (col < 16 && key < a.Lk) part[key] = key < u.L ? x[0] : 0.f;
}

// 16 bits: tiles of 32 query rows (and their LSE) go HBM -> LDS by loads that
// write LDS, three tiles ahead in a ring of four, and tile t + 1's products run
// beside tile t's exponentials.  The ring's slots are LDS objects of their own and
// the loop is unrolled over them, so that the compiler sees that no load in flight
// writes the slot being read; with an index it waits for every load first.
template <typename E, int D>
__global__ __launch_bounds__(256, 2) void key_weights_kernel(KeyWeightArgs a) {
  using T = Bf16Tile<D, 32>;
  constexpr int KB = key_blocks(D), ROWB = T::ROWB;
  constexpr int NLD = 32 / 4 / T::RPI > 0 ? 32 / 4 / T::RPI : 1;  // loads per wave per tile
  static_assert(T::RPI * NLD * 4 == 32, "tile rows");
  __shared__ __attribute__((aligned(1024))) unsigned char qs0[T::TILE_B + 1024], qs1[T::TILE_B + 1024],
      qs2[T::TILE_B + 1024], qs3[T::TILE_B + 1024];  // a tile, then each wave's copy of its LSE
  auto slot = [&](auto i) -> unsigned char* {
    constexpr int I = decltype(i)::value & 3;
    if constexpr (I == 0) return qs0;
    else if constexpr (I == 1) return qs1;
    else if constexpr (I == 2) return qs2;
    else return qs3;
  };
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  int k_first;
  const KeyWork u = key_work(a, 128 * KB, k_first);
  const int k0 = k_first + 32 * KB * w;
  f32x16 acc[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) acc[kb] = f32x16{};
  const int n = (u.q_hi - u.q_lo + 31) / 32;
  if (n > 0) {
    const uint32_t rowstride = (uint32_t)a.Hq * a.rdim * 2;
    const unsigned char* Q = (const unsigned char*)a.q + ((size_t)u.b * a.Lq * a.Hq + u.h) * a.rdim * 2;
    uint32_t voff[NLD];
#pragma unroll
    for (int j = 0; j < NLD; ++j) {
      const int r = 8 * w + T::RPI * j + lane / T::NC, slot = lane % T::NC;
      voff[j] = row_chunk(r, rowstride, slot ^ T::swz_k(r), a.rdim);
    }
    const float* lse = a.lse + ((size_t)u.b * a.Hq + u.h) * a.Lq;
    auto issue = [&](int t, unsigned char* q) {
      const int t0 = u.q_lo + 32 * t;
      // (a tile past the end: empty buffers, so that every path issues the same loads)
      const int rows = max(min(32, u.q_hi - t0), 0);
      const uint32_t bytes = rows > 0 ? (uint32_t)(rows - 1) * rowstride + a.rdim * 2 : 0u;
      const rsrc_t rq = make_rsrc(Q + (size_t)min(t0, a.Lq - 1) * rowstride, bytes);
      const rsrc_t rl = make_rsrc(lse + min(t0, a.Lq - 1), 4 * rows);
#pragma unroll
      for (int j = 0; j < NLD; ++j) buffer_load_lds16(rq, q + (8 * w + T::RPI * j) * ROWB, voff[j]);
      buffer_load_lds4(rl, q + T::TILE_B + 256 * w, 4 * lane);
    };
    typename E::v8 kf[KB][D / 16];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int key = k0 + 32 * kb + col;
      const uint16_t* krow = (const uint16_t*)a.k + (((size_t)u.b * a.Lk + min(key, a.Lk - 1)) * a.G + u.g) * a.rdim;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        u32x4 r = {0u, 0u, 0u, 0u};
        if (key < u.L && 16 * s + 8 * half < a.rdim) r = *(const u32x4*)(krow + 16 * s + 8 * half);
        kf[kb][s] = E::as8(r);
      }
    }
    uint32_t offQ[D / 16];
#pragma unroll
    for (int st = 0; st < D / 16; ++st) offQ[st] = col * ROWB + 16 * ((2 * st + half) ^ T::swz_k(col));
    auto scores = [&](const unsigned char* q, f32x16* s) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) s[kb] = f32x16{};
#pragma unroll
      for (int st = 0; st < D / 16; ++st) {
        const typename E::v8 qf = E::as8(*(const u32x4*)(q + offQ[st]));
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) s[kb] = E::mma32(kf[kb][st], qf, s[kb]);
      }
    };
    // register r of block kb: key k0 + 32 kb + 8 (r / 4) + 4 half + r % 4, query t0 + col
    auto mask = [&](int t, f32x16* s) {
      const int t0 = u.q_lo + 32 * t;
      if (a.causal && k0 + 32 * KB - 1 > t0 + a.shift) {
        asm volatile("");  // (a branch: as selects the comparisons ran on every tile)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const int lim = t0 + col + a.shift - (k0 + 32 * kb + 4 * half);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (8 * (r >> 2) + (r & 3) > lim) s[kb][r] = -INFINITY;
        }
      }
    };
    auto add = [&](f32x16* s, float l2) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[kb][r] += fast_exp2(fmaf(s[kb][r], a.cx, -l2));
    };
    f32x16 sa[KB], sb[KB];
    auto lse_of = [&](int t, const unsigned char* q) {  // in log2 units; +inf: no row, or one without a valid key
      const float l = ((const float*)(q + T::TILE_B + 256 * w))[col];
      return u.q_lo + 32 * t + col < u.q_hi ? l * kLog2e : INFINITY;
    };
    issue(0, qs0);
    issue(1, qs1);
    issue(2, qs2);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    scores(qs0, sa);
    float l = lse_of(0, qs0);
    // Iteration t forms the scores of tile t + 1, which has landed, and loads tile
    // t + 3 into the slot of tile t - 1, last read in iteration t - 2.  Its end waits
    // for tile t + 2, loaded two iterations before it is read.
    auto step = [&](auto i, int t, f32x16* s, f32x16* next) {
      constexpr int I = decltype(i)::value;
      unsigned char* q = slot(std::integral_constant<int, I + 1>{});
      issue(t + 3, slot(std::integral_constant<int, I + 3>{}));
      const float l_next = lse_of(t + 1, q);
      mask(t, s);
      // one basic block from here: the products beside the exponentials
      scores(q, next);
      add(s, l);
      // issue order: the first fragments, then each MFMA with the sums of two scores
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // DS reads
#pragma unroll
      for (int j = 0; j < KB * D / 16; ++j) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
        __builtin_amdgcn_sched_group_barrier(0x402, 768 / D, 0);  // VALU incl. transcendental
        if (j % KB == KB - 1) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      l = l_next;
      wait_vmcnt<NLD + 1>();  // all but tile t + 3's
      stage_barrier();
    };
    for (int t = 0; t < n; t += 4) {
      step(std::integral_constant<int, 0>{}, t, sa, sb);
      if (t + 1 >= n) break;
      step(std::integral_constant<int, 1>{}, t + 1, sb, sa);
      if (t + 2 >= n) break;
      step(std::integral_constant<int, 2>{}, t + 2, sa, sb);
      if (t + 3 >= n) break;
      step(std::integral_constant<int, 3>{}, t + 3, sb, sa);
    }
    wait_vmcnt<0>();  // the last (empty) tiles' loads still write LDS
  }
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) put_weights(a, u, acc[kb], k0 + 32 * kb);
}

__device__ __forceinline__ f32x16 mma_f32(float a, float b, f32x16 c) { return mfma32x32x2f32(a, b, c); }

// float32: the same on v_mfma_f32_32x32x2f32, two features a step.  K's lane
// holds feature half + 2 i of key col in register i.  Bound by the products' rate: 2048
// causal rows of 16 heads over 4 KV heads of 128 107 us, 80 TFLOP/s (121 with tiles
// loaded between two barriers).
template <int D>
__global__ __launch_bounds__(256) void key_weights_f32_kernel(KeyWeightArgs a) {
  constexpr int BQ = 32, LD = D + 4;  // padded rows: 32 lanes reading a feature pair touch distinct banks
  __shared__ __attribute__((aligned(16))) float qs[BQ * LD];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, col = lane & 31, half = lane >> 5;
  int k_first;
  const KeyWork u = key_work(a, 128, k_first);
  const int k0 = k_first + 32 * w;
  f32x16 acc = {};
  if (u.q_lo < u.q_hi) {
    // features 4 i + 2 half .. + 1 of key col: step 2 i contracts 4 i and 4 i + 2
    float2 kf[D / 4];
    const int key = k0 + col;
    const float* krow = (const float*)a.k + (((size_t)u.b * a.Lk + min(key, a.Lk - 1)) * a.G + u.g) * D;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) kf[i] = *(const float2*)(krow + 4 * i + 2 * half);
    if (key >= u.L)
#pragma unroll
      for (int i = 0; i < D / 4; ++i) kf[i] = make_float2(0.f, 0.f);
    const float* lse = a.lse + ((size_t)u.b * a.Hq + u.h) * a.Lq;
    const float* Q = (const float*)a.q + ((size_t)u.b * a.Lq * a.Hq + u.h) * D;
    // The next tile is on its way to registers while this one is worked on.
    constexpr int N = BQ * D / 4 / 256;
    f32x4 x[N];
    float l_raw;
    auto fetch = [&](int t0) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int i = tid + 256 * n, r = min(t0 + i / (D / 4), u.q_hi - 1);
        x[n] = *(const f32x4*)(Q + (size_t)r * a.Hq * D + 4 * (i % (D / 4)));
      }
      l_raw = lse[min(t0 + col, u.q_hi - 1)];
    };
    fetch(u.q_lo);
    for (int t0 = u.q_lo; t0 < u.q_hi; t0 += BQ) {
      __syncthreads();
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int i = tid + 256 * n, r = i / (D / 4);
        *(f32x4*)(qs + r * LD + 4 * (i % (D / 4))) = t0 + r < u.q_hi ? x[n] : f32x4{};
      }
      const float l2 = (t0 + col < u.q_hi ? l_raw : INFINITY) * kLog2e;
      __syncthreads();
      if (t0 + BQ < u.q_hi) fetch(t0 + BQ);
      f32x16 s = {};
#pragma unroll
      for (int i = 0; i < D / 4; ++i) {
        const float2 q2 = *(const float2*)(qs + col * LD + 4 * i + 2 * half);
        s = mma_f32(kf[i].x, q2.x, s);
        s = mma_f32(kf[i].y, q2.y, s);
      }
      if (a.causal && k0 + 31 > t0 + a.shift) {
        const int lim = t0 + col + a.shift - (k0 + 4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (8 * (r >> 2) + (r & 3) > lim) s[r] = -INFINITY;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[r] += fast_exp2(fmaf(s[r], a.cx, -l2));
    }
  }
  put_weights(a, u, acc, k0);
}

// Adds the parts, in their order, to the weights so far.
__global__ __launch_bounds__(256) void add_weights_kernel(const float* part, const float* w_in, float* w_out, int parts,
                                                         int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float x = 0.f;
#pragma unroll 8
    for (int p = 0; p < parts; ++p) x += part[p * n + i];
    w_out[i] = (w_in ? w_in[i] : 0.f) + x;
  }
}

// Splits of the query rows: two workgroups per CU and as many again for the causal
// half that has nothing to do.  (A workgroup first loads the fragments of 256 keys:
// 4096 x 16 heads over 4, causal / full, us: 4 splits 58 / 79, 8 60 / 85, 16 71 / 104.)
static int64_t row_splits(int64_t batch, int64_t q_len, int64_t kv_len, int64_t q_heads) {
  const int64_t blocks = (kv_len + 255) / 256 * batch * q_heads;
  return std::clamp<int64_t>(1024 / std::max<int64_t>(blocks, 1), 1, std::max<int64_t>((q_len + 255) / 256, 1));
}

}  // namespace pjx

using namespace pjx;

extern "C" size_t pjx_weighted_decode_workspace_size(int64_t batch, int64_t kv_heads, int64_t rows, int64_t kv_len,
                                                     int64_t head_dim, int64_t chunk) {
  return partial_bytes(batch, kv_heads, rows, kv_len, head_dim, scored_chunk(batch, kv_heads, kv_len, chunk)) +
         (size_t)(batch * kv_heads * rows * score_stride(kv_len)) * 4;
}

extern "C" int pjx_weighted_decode(int dtype, const void* q, const void* k, const void* v, const int32_t* kv_lengths,
                                   const float* weights, float* weights_out, void* o, float* lse, void* workspace,
                                   size_t workspace_bytes, int64_t batch, int64_t q_len, int64_t kv_len,
                                   int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t row_dim,
                                   const pjx_cache_strides* strides, float sm_scale, int64_t chunk, void* stream) {
  clear_error();
  const char* who = "pjx_weighted_decode";
  DecodeArgs a = {};
  const int rc = fill_cache_decode(a, who, dtype, q, k, v, kv_lengths, o, lse, batch, q_len, kv_len, q_heads, kv_heads,
                                   head_dim, row_dim, strides, sm_scale, scored_chunk(batch, kv_heads, kv_len, chunk));
  if (rc != PJX_OK) return rc;
  const int64_t rows = q_heads / kv_heads * q_len;
  if (rows > kMaxScoredRows) return fail(PJX_ERR_INVALID, "pjx_weighted_decode: at most 64 rows per KV head");
  if (batch == 0) return PJX_OK;
  hipStream_t s = (hipStream_t)stream;
  const bool f32 = dtype == PJX_DTYPE_F32;
  if (kv_len == 0)
    return write_keyless(o, lse, (size_t)(batch * q_len * q_heads * row_dim), f32, (size_t)(batch * q_heads * q_len), s,
                         who);
  if (!weights_out) return fail(PJX_ERR_INVALID, "pjx_weighted_decode: null pointer");
  if (!workspace || workspace_bytes < pjx_weighted_decode_workspace_size(batch, kv_heads, rows, kv_len, head_dim, a.chunk))
    return fail(PJX_ERR_WORKSPACE, "pjx_weighted_decode: workspace missing or too small");
  if ((uintptr_t)workspace % 16) return fail(PJX_ERR_INVALID, "pjx_weighted_decode: the workspace must start on 16 bytes");
  const size_t parts = partial_bytes(batch, kv_heads, rows, kv_len, head_dim, a.chunk);
  a.scores = (float*)((char*)workspace + parts);
  a.score_ld = score_stride(kv_len);
  const int d = (int)head_dim;
  const int nrb = gqa_row_blocks(a.rows, d, d, f32);
  a.rpg = kRows * nrb;
  if (f32)
    return d == 64    ? run_scored_f32<64>(a, nrb, weights, weights_out, workspace, parts, s)
           : d == 128 ? run_scored_f32<128>(a, nrb, weights, weights_out, workspace, parts, s)
                      : run_scored_f32<256>(a, nrb, weights, weights_out, workspace, parts, s);
  return a.f16 ? run_scored_16<F16Fmt>(a, d, nrb, weights, weights_out, workspace, parts, s)
               : run_scored_16<Bf16Fmt>(a, d, nrb, weights, weights_out, workspace, parts, s);
}

extern "C" size_t pjx_key_weights_workspace_size(int64_t batch, int64_t q_len, int64_t kv_len, int64_t q_heads) {
  return (size_t)(batch * q_heads * kv_len * row_splits(batch, q_len, kv_len, q_heads)) * 4;
}

extern "C" int pjx_key_weights(int dtype, const void* q, const void* k, const float* lse, const int32_t* kv_lengths,
                               const float* weights, float* weights_out, void* workspace, size_t workspace_bytes,
                               int64_t batch, int64_t q_len, int64_t kv_len, int64_t q_heads, int64_t kv_heads,
                               int64_t head_dim, int64_t row_dim, int causal, int64_t causal_shift, float sm_scale,
                               void* stream) {
  clear_error();
  char buf[256];
  auto bad = [&](const char* what) {
    snprintf(buf, sizeof(buf), "pjx_key_weights: %s", what);
    return fail(PJX_ERR_INVALID, buf);
  };
  if (dtype != PJX_DTYPE_BF16 && dtype != PJX_DTYPE_F16 && dtype != PJX_DTYPE_F32)
    return bad("dtype must be PJX_DTYPE_BF16, PJX_DTYPE_F16 or PJX_DTYPE_F32");
  const bool f32 = dtype == PJX_DTYPE_F32;
  if (batch < 0 || q_len < 0 || kv_len < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads) return bad("bad sizes");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return bad("head_dim must be 64, 128 or 256");
  if (row_dim != head_dim && (f32 || row_dim <= 0 || row_dim > head_dim || row_dim % 8))
    return bad("row_dim must be head_dim, or in 16 bits a multiple of 8 up to it");
  if (!(sm_scale > 0.f)) return bad("sm_scale must be > 0");
  const int64_t most = (int64_t)1 << 40;
  if (q_len > (1 << 28) || kv_len > (1 << 28) || causal_shift > (1 << 28) || causal_shift < -(1 << 28) ||
      batch * q_heads > (1 << 22) || q_heads * row_dim > (1 << 24) || batch * q_heads * std::max(q_len, kv_len) > most / head_dim)
    return bad("sizes out of range");
  if (batch * kv_len == 0) return PJX_OK;
  if (!weights_out || !k || (q_len > 0 && (!q || !lse))) return bad("null pointer");
  if (((uintptr_t)q | (uintptr_t)k) % 16) return bad("q and k must start on 16 bytes");
  if (!workspace || workspace_bytes < pjx_key_weights_workspace_size(batch, q_len, kv_len, q_heads))
    return fail(PJX_ERR_WORKSPACE, "pjx_key_weights: workspace missing or too small");
  KeyWeightArgs a = {};
  a.q = q; a.k = k; a.lse = lse; a.lengths = kv_lengths; a.part = (float*)workspace;
  a.B = (int)batch; a.Lq = (int)q_len; a.Lk = (int)kv_len; a.Hq = (int)q_heads; a.G = (int)kv_heads;
  a.rdim = (int)row_dim;
  a.causal = causal != 0;
  a.shift = (int)causal_shift;
  a.splits = (int)row_splits(batch, q_len, kv_len, q_heads);
  a.q_step = (int)(((q_len + a.splits - 1) / a.splits + 31) / 32 * 32);
  a.cx = sm_scale * kLog2e;
  const int64_t units = batch * q_heads * a.splits, per = f32 ? 128 : 128 * key_blocks((int)head_dim),
                groups = (kv_len + per - 1) / per;
  if (units * groups > 0xffffffffLL / 256) return bad("sizes out of range");
  hipStream_t s = (hipStream_t)stream;
  const dim3 grid((unsigned)(units * groups)), block(256);
  if (f32) {
    if (head_dim == 64) launch_kernel<key_weights_f32_kernel<64>>(grid, block, 0, s, a);
    else if (head_dim == 128) launch_kernel<key_weights_f32_kernel<128>>(grid, block, 0, s, a);
    else launch_kernel<key_weights_f32_kernel<256>>(grid, block, 0, s, a);
  } else if (dtype == PJX_DTYPE_F16) {
    if (head_dim == 64) launch_kernel<key_weights_kernel<F16Fmt, 64>>(grid, block, 0, s, a);
    else if (head_dim == 128) launch_kernel<key_weights_kernel<F16Fmt, 128>>(grid, block, 0, s, a);
    else launch_kernel<key_weights_kernel<F16Fmt, 256>>(grid, block, 0, s, a);
  } else {
    if (head_dim == 64) launch_kernel<key_weights_kernel<Bf16Fmt, 64>>(grid, block, 0, s, a);
    else if (head_dim == 128) launch_kernel<key_weights_kernel<Bf16Fmt, 128>>(grid, block, 0, s, a);
    else launch_kernel<key_weights_kernel<Bf16Fmt, 256>>(grid, block, 0, s, a);
  }
  const int rc = check_launch("pjx_key_weights");
  if (rc != PJX_OK) return rc;
  const int64_t n = batch * kv_heads * kv_len;
  launch_kernel<add_weights_kernel>(dim3((unsigned)std::min<int64_t>((n + 255) / 256, 65536)), block, 0, s,
                                    (const float*)a.part, weights, weights_out, (int)(q_heads / kv_heads * a.splits), n);
  return check_launch("pjx_key_weights");
}
