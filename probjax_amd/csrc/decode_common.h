// What the split-KV decode kernels share: the arguments, the schedule of the
// work items, the combine of a workgroup's waves, and the GQA decode itself
// (16-bit and fp32), which three kernel families instantiate:
//   kPlain   decode over a cache (decode.hip)
//   kTree    drafted tokens that form a tree, over a cache (tree_decode.hip)
//   kScores  decode that keeps its scores for the keys' weights (key_weights.hip)
#pragma once

#include <type_traits>

#include "pjx_common.h"
#include "pjx_internal.h"

namespace pjx {

constexpr int kDecThreads = 256;
constexpr int kTile = 64;       // keys per latent tile (16 per wave)
constexpr int kRows = 16;       // query rows per MFMA column block

// Kernel family of a GQA decode instance.
constexpr int kPlain = 0, kTree = 1, kScores = 2;

struct DecodeArgs {
  const uint16_t* q;   // bf16 / fp16 (fp32 decode: the same pointers hold floats)
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* lengths;
  uint16_t* o;         // 16-bit output (bf16, or fp16 when f16), or null with o32
  float* o32;          // fp32 output of the fp32 decode, else null
  int f16;             // 16-bit inputs and output are fp16 (else bf16)
  float* lse;
  float* ws_o;   // [B*G][nch][rows][dv] unnormalised partial outputs
  float* ws_ml;  // [B*G][nch][rows][2]  running max (log2 units), sum
  int B, Lq, Lk, Hq, G, rows;
  int fold;      // 1: row = t*H + h (MLA); 0: row = gi*Lq + t (GQA)
  int chunk, nch;
  int dv;        // output dims of the kernel (the partials' row)
  int orow;      // elements of an output row in memory (0: dv), and of q, k and v rows in the rows kernels
  float cx;      // sm_scale * log2(e)
  // kTree and kScores: elements between consecutive sequences, tokens and heads
  // of the caches.
  int64_t k_b, k_t, k_h, v_b, v_t, v_h;
  // kTree: `extra` drafted tokens (Lq of them) whose keys lie behind the
  // sequence's prefix; their parents, or a byte matrix of what each sees, with
  // tree_step elements between sequences (0: one tree for all).
  int extra;
  const int32_t* parents;
  const uint8_t* tree_mask;
  int64_t tree_step;
  // kScores: s * cx of every row and key, [B*G][rows][score_ld].
  float* scores;
  int64_t score_ld;
  // Query rows per row group: the rows of a KV head are split into groups of
  // `rpg` (16 per MFMA column block of the kernel), one per blockIdx.y; each
  // group's workgroups stream the same keys.
  int rpg;
};

__device__ __forceinline__ void row_to_head(const DecodeArgs& a, int g, int r, int& t, int& h) {
  if (a.fold) {
    t = r / a.Hq;
    h = r % a.Hq;
  } else {
    const int per = a.Hq / a.G;
    t = r % a.Lq;
    h = g * per + r / a.Lq;
  }
}

// Keys of sequence b that the lengths name (kTree: its prefix), and all of its
// keys (with the drafted tokens', as far as the cache reaches).
__device__ __forceinline__ int prefix_len(const DecodeArgs& a, int b) {
  int L = a.Lk - a.extra;
  if (a.lengths) L = min(a.Lk, max(a.lengths[b], 0));
  return L;
}
__device__ __forceinline__ int seq_len(const DecodeArgs& a, int b) {
  return min(a.Lk, prefix_len(a, b) + a.extra);
}

// ---------------------------------------------------------------------------
// Drafted tokens (kTree).  bits[t] holds what token t sees of the drafted keys.
// ---------------------------------------------------------------------------
constexpr int kTreeMax = 256;              // drafted tokens
constexpr int kTreeWords = kTreeMax / 32;  // words of a token's set
struct TreeTable {
  uint32_t bits[kTreeMax][kTreeWords];
  int jump[kTreeMax];
};
static_assert(kTreeMax <= kDecThreads, "one thread per token");

// Fills the table; every thread of a workgroup of WAVES waves calls it.  From
// parents: each token's set starts as itself and every round adds the set of
// the token it jumps to while the jumps double in length, so a chain of T
// tokens takes log2(T) rounds; up to 64 tokens by one wave between its lanes
// (26 tokens: 2.1 us with a barrier after every round).  A parent that is no
// earlier token ends a chain.
template <int WAVES>
__device__ __forceinline__ void build_tree(const DecodeArgs& a, int b, TreeTable& tt) {
  const int tid = threadIdx.x, lane = tid & 63, T = a.Lq;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (a.parents && T <= 64) {
    if (wave == 0) {
      const int p = a.parents[(size_t)b * a.tree_step + min(lane, T - 1)];
      int jump = p < lane ? p : -1;
      uint32_t lo = lane < 32 ? 1u << lane : 0u, hi = lane < 32 ? 0u : 1u << (lane - 32);
      for (int span = 1; span < T; span *= 2) {
        const int src = max(jump, 0), next = __shfl(jump, src);
        const uint32_t more_lo = __shfl(lo, src), more_hi = __shfl(hi, src);
        if (jump >= 0) {
          lo |= more_lo;
          hi |= more_hi;
          jump = next;
        }
      }
#pragma unroll
      for (int w = 0; w < kTreeWords; ++w)
        if (lane < T) tt.bits[lane][w] = w == 0 ? lo : w == 1 ? hi : 0u;
    }
  } else if (a.parents) {
    if (tid < T) {
      const int p = a.parents[(size_t)b * a.tree_step + tid];
      tt.jump[tid] = p < tid ? p : -1;
#pragma unroll
      for (int w = 0; w < kTreeWords; ++w) tt.bits[tid][w] = w == tid >> 5 ? 1u << (tid & 31) : 0u;
    }
    __syncthreads();
    for (int span = 1; span < T; span *= 2) {
      uint32_t add[kTreeWords] = {};
      int next = -1;
      if (tid < T) {
        const int j = tt.jump[tid];
        if (j >= 0) {
          next = tt.jump[j];
#pragma unroll
          for (int w = 0; w < kTreeWords; ++w) add[w] = tt.bits[j][w];
        }
      }
      __syncthreads();
      if (tid < T) {
        tt.jump[tid] = next;
#pragma unroll
        for (int w = 0; w < kTreeWords; ++w) tt.bits[tid][w] |= add[w];
      }
      __syncthreads();
    }
  } else {
    // 64 bytes of a row a time, the loads of 8 rows issued before the first is used
    const uint8_t* m = a.tree_mask + (size_t)b * a.tree_step;
    for (int j0 = 0; j0 < T; j0 += 64) {
      const int j = min(j0 + lane, T - 1);
      const bool in = j0 + lane < T;
      for (int t0 = wave; t0 < T; t0 += 8 * WAVES) {
        uint8_t x[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = m[min(t0 + u * WAVES, T - 1) * T + j];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int t = t0 + u * WAVES;
          const uint64_t seen = __builtin_amdgcn_ballot_w64(in & (x[u] != 0));
          if (lane == 0 && t < T) {
            tt.bits[t][j0 >> 5] = (uint32_t)seen;
            tt.bits[t][(j0 >> 5) + 1] = (uint32_t)(seen >> 32);
          }
        }
      }
    }
  }
  __syncthreads();
}

// Whether token t sees the key `j` slots behind the prefix's end (j < 0: a key
// of the prefix, which every token sees).
__device__ __forceinline__ bool tree_sees(const TreeTable& tt, int T, int t, int j) {
  return j < 0 || (j < T && ((tt.bits[t][j >> 5] >> (j & 31)) & 1u));
}

// Whether slot t of sequence b holds a token (a parent below -1: none).
__device__ __forceinline__ bool tree_token(const DecodeArgs& a, int b, int t) {
  return !a.parents || a.parents[(size_t)b * a.tree_step + t] >= -1;
}

// The bits of a float for a test that NaN takes part in.  They pass through an
// empty asm: the sources are compiled without NaN in mind, and a test of a
// float's bits is otherwise recognised as one of the float and NaN ruled out.
__device__ __forceinline__ uint32_t plain_bits(float x) {
  uint32_t u = __float_as_uint(x);
  asm volatile("" : "+v"(u));
  return u;
}
// Whether a float's bits are those of an infinity or NaN.
__device__ __forceinline__ bool not_finite(uint32_t u) { return (u & 0x7f800000u) == 0x7f800000u; }

// 16-bit elements of a dword whose exponent is all ones (infinities, NaN) -> 0.
template <typename E>
__device__ __forceinline__ uint32_t finite_halves(uint32_t x) {
  constexpr uint32_t ex = E::kF16 ? 0x7c00u : 0x7f80u;
  if ((x & ex) == ex) x &= 0xffff0000u;
  if ((x & (ex << 16)) == ex << 16) x &= 0xffffu;
  return x;
}

// Keeps the compiler from moving LDS accesses of one wave across this point;
// the LDS itself executes one wave's accesses in program order.
__device__ __forceinline__ void wave_lds_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Whether a row with this sum of weights has a valid key (a NaN sum: yes).
__device__ __forceinline__ bool some_key(float sum) { return plain_bits(sum) != 0u; }

// Writes 4 consecutive dims d..d+3 (d a multiple of 4) of one work item's combined
// result: the final output and LSE when the item covers the whole sequence, else
// the unnormalised partial (O relative to max M, plus M and the sum) for the merge
// kernel.  (kPlain promises no alignment of a final output.)
template <int X>
__device__ __forceinline__ void emit_row(const DecodeArgs& a, int b, int g, int r, int d, size_t part, bool final_out,
                                         float M, float Ls, f32x4 O) {
  if (final_out) {
    int t, h;
    row_to_head(a, g, r, t, h);
    const bool some = X == kPlain ? Ls > 0.f : some_key(Ls);
    f32x4 out;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = some ? O[e] / Ls : 0.f;
    const size_t oi = ((size_t)(b * a.Lq + t) * a.Hq + h) * a.orow + d;
    if constexpr (X == kPlain) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (a.o32)
          a.o32[oi + e] = out[e];
        else
          a.o[oi + e] = a.f16 ? F16Fmt::bits(out[e]) : Bf16Fmt::bits(out[e]);
      }
    } else if (a.o32) {
      *(f32x4*)(a.o32 + oi) = out;
    } else {
      *(u32x2*)(a.o + oi) = a.f16 ? u32x2{F16Fmt::pack2(out[0], out[1]), F16Fmt::pack2(out[2], out[3])}
                                  : u32x2{Bf16Fmt::pack2(out[0], out[1]), Bf16Fmt::pack2(out[2], out[3])};
    }
    if (a.lse && d == 0)
      a.lse[((size_t)b * a.Hq + h) * a.Lq + t] = some ? (M + __log2f(Ls)) * kLn2 : INFINITY;
  } else {
    *(f32x4*)(a.ws_o + (part * a.rows + r) * a.dv + d) = O;
    if (d == 0) {
      a.ws_ml[(part * a.rows + r) * 2] = M;
      a.ws_ml[(part * a.rows + r) * 2 + 1] = Ls;
    }
  }
}

// Work item `item` of a decode: (batch b, kv group g, chunk chunk_id).
// The hardware starts workgroups in index order as slots free up, so the
// index order is the schedule.  With per-sequence lengths (B <=
// kSchedMaxBatch) the items run longest first: every full chunk (sequence by
// sequence, or chunk-major where every sequence has as many), then each
// sequence's partial last chunk in decreasing size, then
// the empty items, which exit at once.  The plain chunk-major order scatters
// the partial chunks through the grid and leaves a tail of full chunks that
// start late.  Every thread calls this (it holds two barriers); L receives
// the sequence's clamped length; false: the item has no keys.
constexpr int kSchedMaxBatch = 256;
static_assert(kSchedMaxBatch <= kDecThreads, "one length per thread");
__device__ bool decode_item(const DecodeArgs& a, int* sched, int& b, int& g, int& chunk_id, int& L, unsigned item) {
  if (!a.lengths || a.B > kSchedMaxBatch) {
    const int BG = a.B * a.G;
    chunk_id = item / BG;
    const int bg = item % BG;
    b = bg / a.G;
    g = bg % a.G;
    L = seq_len(a, b);
    return chunk_id * a.chunk < L;
  }
  const int q = item / a.G, t = threadIdx.x;
  g = item % a.G;
  int* nfs = sched + 4;                 // full chunks per sequence
  int* rms = nfs + kSchedMaxBatch;      // keys of the partial last chunk
  int Lt = 0, nf = 0, rt = 0;
  if (t < a.B) {
    Lt = seq_len(a, t);
    nf = Lt / a.chunk;
    rt = Lt - nf * a.chunk;
    nfs[t] = nf;
    rms[t] = rt;
  }
  if (t == 0) sched[0] = -1;
  __syncthreads();
  if (t < a.B) {
    // sequence t: its full chunks are rows [pre, pre + nf) of the full part;
    // its partial chunk (rt > 0) has the rank of rt among the partial chunks
    // (ties by sequence index)
    int pre = 0, full = 0, rank = 0, nf_min = nf, nf_max = nf;
#pragma unroll 8
    for (int u = 0; u < a.B; ++u) {
      const int nu = nfs[u], ru = rms[u];
      full += nu;
      pre += u < t ? nu : 0;
      nf_min = min(nf_min, nu);
      nf_max = max(nf_max, nu);
      rank += (ru > 0 && (ru > rt || (ru == rt && u < t))) ? 1 : 0;
    }
    int c = -1;
    if (nf_min == nf_max) {
      // as many full chunks in every sequence: chunk-major, as without lengths
      if (q < full && q % a.B == t) c = q / a.B;
    } else if (q >= pre && q < pre + nf) {
      c = q - pre;
    }
    if (rt > 0 && q >= full && q - full == rank) c = nf;
    if (c >= 0) {
      sched[0] = t;
      sched[1] = c;
      sched[2] = Lt;
    }
  }
  __syncthreads();
  b = sched[0];
  chunk_id = sched[1];
  L = sched[2];
  if (b < 0) {
    b = 0;
    L = 0;
    return false;
  }
  return true;
}

// emit_row of the latent decode, whose outputs are products with 1 / sum.
__device__ __forceinline__ void emit_row_quad(const DecodeArgs& a, int b, int g, int r, int d,
                                              size_t part, bool final_out, float M, float Ls,
                                              f32x4 O) {
  if (final_out) {
    int t, h;
    row_to_head(a, g, r, t, h);
    const float inv = Ls > 0.f ? 1.f / Ls : 0.f;
    const size_t oi = ((size_t)(b * a.Lq + t) * a.Hq + h) * a.orow + d;
    if (a.o32) {
      *(f32x4*)(a.o32 + oi) = O * inv;
    } else {
      const u32x2 pk = a.f16 ? u32x2{F16Fmt::pack2(O[0] * inv, O[1] * inv), F16Fmt::pack2(O[2] * inv, O[3] * inv)}
                             : u32x2{Bf16Fmt::pack2(O[0] * inv, O[1] * inv), Bf16Fmt::pack2(O[2] * inv, O[3] * inv)};
      *(u32x2*)(a.o + oi) = pk;
    }
    if (a.lse && d == 0)
      a.lse[((size_t)b * a.Hq + h) * a.Lq + t] = Ls > 0.f ? (M + __log2f(Ls)) * kLn2 : INFINITY;
  } else {
    *(f32x4*)(a.ws_o + (part * a.rows + r) * a.dv + d) = O;
    if (d == 0) {
      a.ws_ml[(part * a.rows + r) * 2] = M;
      a.ws_ml[(part * a.rows + r) * 2 + 1] = Ls;
    }
  }
}

// ---------------------------------------------------------------------------
// GQA split-KV decode.  One workgroup = one (chunk, batch, kv group) work
// item; its 4 waves split the chunk's keys into contiguous quarters and run
// independent online softmaxes (no block barrier inside the key loop), then
// combine their (max, sum, O) in LDS.  The rows = (Hq/Hkv)*Lq query rows of
// the KV head are NRB blocks of 16 MFMA columns (up to 64 rows, the
// reference's largest packed tile, attention_splitkv.py:155-170).  Per
// iteration a wave takes 32 keys:
//   * K rows are loaded straight into the A operand of
//     v_mfma_f32_16x16x32_bf16 (lane: key l%16, 16 bytes of dims), S^T = K Q^T
//     for each row block;
//   * V rows are loaded 4 keys x 8 dims per lane, packed with v_perm into
//     [dim][key] order and written to a wave-private LDS slab, from which the
//     A operand of O^T += V^T P^T is two 8-byte reads, shared by the row
//     blocks;
//   * the next iteration's K and V loads are issued before this iteration's
//     softmax and P.V, so HBM traffic overlaps the arithmetic.
// Keys at or past the sequence length are never read.
// ---------------------------------------------------------------------------

// Combines the 4 waves' (max, sum, O^T) of row block rb through LDS scratch
// red (>= 4 x 16 x D floats + 4 x 16 x 2) and emits rows row0 + 16rb .. of the
// item (D = the output dims).  acc[i] holds quad quad_of(i) of row
// row0 + 16rb + c16 of O, a quad being 4 consecutive dims.  Rows lie in quads of dims, quad c of row r at c ^ r, so that
// neither the writes (16 rows at once) nor the reads (a row at once) meet in a bank,
// and each thread combines a quad (32 rows of 128 element by element: 7 us of the 17
// of a float32 work item).
template <int D, int X, typename Q>
__device__ __forceinline__ void combine_rows(const DecodeArgs& a, float* red, const f32x4* acc, Q quad_of,
                                             float m_run, float l_run, int row0, int rb, int b, int g,
                                             size_t part, bool final_out) {
  static_assert(D % 64 == 0, "16 quads or more");
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int c16 = lane & 15, q4 = lane >> 4;
  float* red_o = red;                  // [4][16 rows][D]
  float* red_ml = red_o + 4 * 16 * D;  // [4][16 rows][2]
  __syncthreads();  // the scratch is free (every wave is done with it)
#pragma unroll
  for (int db = 0; db < D / 16; ++db)
    *(f32x4*)(red_o + (w * 16 + c16) * D + 4 * (quad_of(db) ^ c16)) = acc[db];
  if (q4 == 0) *(float2*)(red_ml + (w * 16 + c16) * 2) = make_float2(m_run, l_run);
  __syncthreads();
  const int nr = min(16, a.rows - row0 - 16 * rb);
  for (int e = tid; e < nr * (D / 4); e += 256) {
    const int r = e / (D / 4), c = e % (D / 4), d = 4 * c;
    if (d >= a.orow) continue;
    float2 ml[4];
    float M = kMaxInit;
#pragma unroll
    for (int ww = 0; ww < 4; ++ww) {
      ml[ww] = *(const float2*)(red_ml + (ww * 16 + r) * 2);
      M = fmaxf(M, ml[ww].x);
    }
    float Ls = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ww = 0; ww < 4; ++ww) {
      const float wt = fast_exp2(ml[ww].x - M);
      Ls = fmaf(wt, ml[ww].y, Ls);
      const f32x4 o = *(const f32x4*)(red_o + (ww * 16 + r) * D + 4 * (c ^ r));
#pragma unroll
      for (int i = 0; i < 4; ++i) O[i] = fmaf(wt, o[i], O[i]);
    }
    if constexpr (X == kTree)
      if (!some_key(Ls)) O = f32x4{0.f, 0.f, 0.f, 0.f};  // a row without a valid key
    emit_row<X>(a, b, g, row0 + 16 * rb + r, d, part, final_out, M, Ls, O);
    if constexpr (X == kScores) {  // the weights' kernel reads every item's statistics
      if (final_out && d == 0) {
        a.ws_ml[(part * a.rows + row0 + 16 * rb + r) * 2] = M;
        a.ws_ml[(part * a.rows + row0 + 16 * rb + r) * 2 + 1] = Ls;
      }
    }
  }
}

// kTree: adds p * v for the infinite and NaN elements v of a 32-key step's V
// rows to the rows that see the key; v_at(key, db, odd) gives the lane's 4 elements
// of output block db and the mask of such ones.
// s holds the step's p (lane layout of S^T), px 512 floats of this wave.
template <int NRB, int NDB, typename V>
__device__ __forceinline__ void add_unbounded(const DecodeArgs& a, const TreeTable& tree, float* px,
                                              const f32x4 (*s)[2], f32x4 (*acc)[NDB], const int* tok, int k0, int w1,
                                              int P, V v_at) {
  const int lane = threadIdx.x & 63, c16 = lane & 15, q4 = lane >> 4;
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb) {
    wave_lds_sync();
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int r = 0; r < 4; ++r) px[(16 * kb + 4 * q4 + r) * 16 + c16] = s[rb][kb][r];
    wave_lds_sync();
#pragma unroll 1
    for (int i = 0; i < min(32, w1 - k0); ++i) {
      const float p = px[16 * i + c16];
      const bool sees = tree_sees(tree, a.Lq, tok[rb], k0 + i - P);
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        int odd = 0;
        const f32x4 v = v_at(k0 + i, db, odd);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (sees && (odd >> e & 1)) acc[rb][db][e] = fmaf(p, v[e], acc[rb][db][e]);
      }
    }
  }
  wave_lds_sync();
}

// Two workgroups per CU where the registers allow it: 16- or 32-row groups at
// head dims up to 128.
template <int D, int DV, int NRB>
constexpr int decode_occupancy() { return (NRB == 4 || D > 128 || DV > 128) ? 1 : 2; }

// ROWS: q, k, v and o rows hold a.orow elements (a multiple of 8, below D = DV)
// and the lanes whose chunk lies past a row's end hold zeros instead of loading.
template <typename E, int D, int DV, int NRB, bool STREAM, bool ROWS, int X = kPlain>
__device__ __forceinline__ void gqa_decode(const DecodeArgs& a) {
  constexpr int KSTEPS = D / 32;  // 32-dim MFMA k-steps of Q.K
  constexpr int NDB = DV / 16;    // 16-dim output blocks
  constexpr int DC = DV / 8;      // 16-byte chunks per V row
  constexpr int VU = DV / 64;     // (4 keys x 8 dims) V units per lane per 32 keys
  constexpr int CR = D / 8;       // 16-byte chunks per K row
  static_assert(!(ROWS && STREAM), "rows of any length take ordinary loads");
  constexpr int KLD = D / 16;     // K chunks per lane per 32-key step (32 * CR / 64 = 2 * KSTEPS)
  static_assert(D % 64 == 0 && DV % 64 == 0, "head dims");
  // Each wave's V^T tile: DV rows (output dims) of the step's 32 keys, 64
  // bytes each, 4 rows to a 256-byte bank line (see vt_at); the same memory
  // then holds the 4 waves' partial rows for the combine.
  constexpr int VT_B = 4 * DV * 64, COMB_B = 4 * 16 * DV * 4 + 4 * 16 * 2 * 4;
  __shared__ __attribute__((aligned(256))) uint16_t vt_lds[(VT_B > COMB_B ? VT_B : COMB_B) / 2];
  __shared__ __attribute__((aligned(16))) uint16_t k_lds[STREAM ? 4 * 32 * D : 8];  // per wave: 32 key rows
  // STREAM: chunk swizzle of K row r in the wave's K slab, a bijection of the
  // row's 16-byte chunks that sends the same chunk of 16 consecutive rows to
  // 16 different bank groups (rows of 128, 256 or 512 bytes)
  auto kswz = [](int r) { return CR >= 16 ? (r & 15) : ((r >> 1) & (CR - 1)); };
  // STREAM: K/V are read once per call, past what the 256 MB MALL holds, with
  // non-temporal loads (measured on this layout: ~7.0 TB/s with full 128-byte
  // lines, against ~5.9 TB/s for ordinary loads)
  auto ld16 = [](const uint16_t* p) -> u32x4 {
    if constexpr (STREAM) return __builtin_nontemporal_load((const u32x4*)p);
    else return *(const u32x4*)p;
  };

  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int c16 = lane & 15, q4 = lane >> 4;
  __shared__ int sched[4 + 2 * kSchedMaxBatch];
  int b, g, chunk_id, L;
  if (!decode_item(a, sched, b, g, chunk_id, L, blockIdx.x)) return;  // nothing past the length is read
  const int bg = b * a.G + g;
  const int c0 = chunk_id * a.chunk;
  // the item's keys split evenly over the 4 waves (32-key steps), so a
  // partial chunk takes a quarter of its length, not up to a full quarter
  // chunk on one wave
  const int per_wave = ((min(L - c0, a.chunk) + 127) >> 7) << 5;
  const int w0 = c0 + w * per_wave;
  const int w1 = min(w0 + per_wave, L);

  const int row0 = blockIdx.y * 16 * NRB;  // this row group's first row
  // kTree: the sequence's prefix; every step that reaches past it asks the
  // table which rows see its drafted keys
  const int P = X == kTree ? prefix_len(a, b) : 0;
  __shared__ typename std::conditional<X == kTree, TreeTable, int>::type tree;
  __shared__ float tree_p[X == kTree ? 4 * 512 : 1];
  int tok[NRB];
  bool has[NRB];  // kTree: the row's slot holds a token
  const int rd = ROWS ? a.orow : D, rdv = ROWS ? a.orow : DV;
  typename E::v8 qf[NRB][KSTEPS];
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb) {
    const int row = row0 + 16 * rb + c16;
    const bool rv = row < a.rows;
    int t = 0, h = 0;
    if (rv) row_to_head(a, g, row, t, h);
    tok[rb] = t;
    has[rb] = X != kTree || tree_token(a, b, t);
    const uint16_t* qrow = a.q + ((size_t)(b * a.Lq + t) * a.Hq + h) * rd;
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      u32x4 r = {0u, 0u, 0u, 0u};
      if (rv && (!ROWS || 32 * s + 8 * q4 < rd)) r = *(const u32x4*)(qrow + 32 * s + 8 * q4);
      qf[rb][s] = E::as8(r);
    }
  }
  const size_t k_tok = X == kPlain ? (size_t)a.G * rd : (size_t)a.k_t;
  const size_t v_tok = X == kPlain ? (size_t)a.G * rdv : (size_t)a.v_t;
  const uint16_t* Kb = a.k + (X == kPlain ? ((size_t)b * a.Lk * a.G + g) * rd : (size_t)(b * a.k_b + g * a.k_h));
  const uint16_t* Vb = a.v + (X == kPlain ? ((size_t)b * a.Lk * a.G + g) * rdv : (size_t)(b * a.v_b + g * a.v_h));
  uint16_t* vl = vt_lds + w * DV * 32;
  // Element offset of 8-byte unit u (keys 4u .. 4u+3) of V^T row r.  The 32
  // units of a 256-byte line (rows 4L .. 4L+3) are XOR-swizzled by F(L) so
  // that both access patterns are free of bank conflicts: the writes of 16
  // lanes (one LDS cycle for ds_write_b64) put one unit of rows 8*dc + e,
  // dc = 0..15, in 16 different lines, whose F values all differ; the reads
  // of 32 lanes (one cycle for ds_read_b64) take units u, u+1 of 16
  // consecutive rows, 4 lines whose F values differ in bits 1-2.
  auto vt_at = [](int row, int unit) {
    const int L = row >> 2;
    const int F = ((L & 3) << 1) | (((L >> 2) & 3) << 3) | ((L >> 4) & 1);
    return 128 * L + 4 * ((8 * (row & 3) + unit) ^ F);
  };

  f32x4 acc[NRB][NDB];
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb)
#pragma unroll
    for (int i = 0; i < NDB; ++i) acc[rb][i] = f32x4{};
  float m_run[NRB], l_run[NRB];
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb) {
    m_run[rb] = kMaxInit;
    l_run[rb] = 0.f;
  }

  // K: without STREAM, loaded straight into the A operand (kr[kb * KSTEPS + s]
  // holds 16 bytes of key 16*kb + c16 at dims 32*s + 8*q4: each load covers
  // 64 bytes of 16 rows).  With STREAM, rows are loaded whole (CR consecutive
  // lanes per row, full 128-byte lines, which non-temporal loads need) into
  // kr[i] = chunk u % CR of row u / CR, u = lane + 64*i, and staged through
  // the wave's K slab, chunk c of row r at c ^ kswz(r).
  u32x4 kr[KLD];
  u32x4 vr[VU][4];
  uint16_t* kl = k_lds + (STREAM ? w * 32 * D : 0);
  auto load_k = [&](int k0) {
    if constexpr (STREAM) {
#pragma unroll
      for (int i = 0; i < KLD; ++i) {
        const int u = lane + 64 * i, key = k0 + u / CR;
        u32x4 r = {0u, 0u, 0u, 0u};
        if (key < w1) r = ld16(Kb + (size_t)key * k_tok + 8 * (u % CR));
        kr[i] = r;
      }
    } else {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int key = k0 + 16 * kb + c16;
        const bool ok = key < w1;
        const uint16_t* p = Kb + (size_t)(ok ? key : 0) * k_tok + 8 * q4;
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) {
          u32x4 r = {0u, 0u, 0u, 0u};
          if (ok && (!ROWS || 32 * s + 8 * q4 < rd)) r = *(const u32x4*)(p + 32 * s);
          kr[kb * KSTEPS + s] = r;
        }
      }
    }
  };
  auto store_k = [&]() {
#pragma unroll
    for (int i = 0; i < KLD; ++i) {
      const int u = lane + 64 * i, row = u / CR;
      *(u32x4*)(kl + row * D + 8 * ((u % CR) ^ kswz(row))) = kr[i];
    }
  };
  auto load_v = [&](int k0) {
#pragma unroll
    for (int i = 0; i < VU; ++i) {
      const int u = lane + 64 * i;
      const int dc = u % DC, kq = u / DC;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = k0 + 4 * kq + j;
        u32x4 r = {0u, 0u, 0u, 0u};
        if (key < w1 && (!ROWS || 8 * dc < rdv)) r = ld16(Vb + (size_t)key * v_tok + 8 * dc);
        vr[i][j] = r;
      }
    }
  };
  auto store_vt = [&]() {
#pragma unroll
    for (int i = 0; i < VU; ++i) {
      const int u = lane + 64 * i;
      const int dc = u % DC, kq = u / DC;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int dw = e >> 1;
        u32x2 pk;
        if (e & 1) {
          pk[0] = pack_hi_halves(vr[i][0][dw], vr[i][1][dw]);
          pk[1] = pack_hi_halves(vr[i][2][dw], vr[i][3][dw]);
        } else {
          pk[0] = pack_lo_halves(vr[i][0][dw], vr[i][1][dw]);
          pk[1] = pack_lo_halves(vr[i][2][dw], vr[i][3][dw]);
        }
        *(u32x2*)(vl + vt_at(8 * dc + e, kq)) = pk;
      }
    }
  };

  // kScores: a step's scores are stored in the next one, before its loads: the
  // wait for the loads then finds the stores done too (both count in order), and
  // not just issued.
  f32x4 scored[X == kScores ? NRB : 1][2];
  auto store_scores = [&](int k0) {
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
      const int row = row0 + 16 * rb + c16;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int key = k0 + 16 * kb + 4 * q4;
        if (row < a.rows && key < w1)
          *(f32x4*)(a.scores + ((size_t)bg * a.rows + row) * a.score_ld + key) = scored[X == kScores ? rb : 0][kb];
      }
    }
  };
  if (w0 < w1) {
    load_k(w0);
    load_v(w0);
  }
  if constexpr (X == kTree) {
    if (c0 + a.chunk > P) build_tree<kDecThreads / 64>(a, b, tree);
  }
  for (int k0 = w0; k0 < w1; k0 += 32) {
    const int kn = k0 + 32;
    // An infinity or NaN in the V row of a drafted key must not reach the rows
    // that do not see it (0 * inf): such elements enter the products as zeros
    // and are added to the rows that see them one by one (add_unbounded).
    bool unbounded = false;
    if constexpr (X == kTree) {
      if (kn > P) {
        uint32_t odd = 0;
#pragma unroll
        for (int i = 0; i < VU; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t x = finite_halves<E>(vr[i][j][e]);
              odd |= x ^ vr[i][j][e];
              vr[i][j][e] = x;
            }
        unbounded = wave_any(odd != 0u);
      }
    }
    store_vt();
    if constexpr (STREAM) {
      store_k();
      wave_lds_sync();
      if constexpr (X == kScores)
        if (k0 > w0) store_scores(k0 - 32);
      if (kn < w1) {
        load_v(kn);
        load_k(kn);
      }
    } else {
      if constexpr (X == kScores)
        if (k0 > w0) store_scores(k0 - 32);
      if (kn < w1) load_v(kn);
    }
    // S^T for keys k0 + 16*kb + 4*q4 + r (register r), query row 16rb + c16;
    // the A operand of k-step st: dims 32*st + 8*q4 of key 16*kb + c16.
    f32x4 s[NRB][2];
    if constexpr (STREAM) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int row = 16 * kb + c16;
#pragma unroll
        for (int st = 0; st < KSTEPS; ++st) {
          const u32x4 kf = *(const u32x4*)(kl + row * D + 8 * ((4 * st + q4) ^ kswz(row)));
#pragma unroll
          for (int rb = 0; rb < NRB; ++rb)
            s[rb][kb] = E::mma16(E::as8(kf), qf[rb][st], st == 0 ? f32x4{} : s[rb][kb]);
        }
      }
    } else {
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          s[rb][kb] = f32x4{};
#pragma unroll
          for (int st = 0; st < KSTEPS; ++st)
            s[rb][kb] = E::mma16(E::as8(kr[kb * KSTEPS + st]), qf[rb][st], s[rb][kb]);
        }
    }
    if constexpr (!STREAM)
      if (kn < w1) load_k(kn);
    if (kn > w1) {
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (k0 + 16 * kb + 4 * q4 + r >= w1) s[rb][kb][r] = -INFINITY;
    }
    if constexpr (X == kTree) {
      if (kn > P) {
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb)
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!tree_sees(tree, a.Lq, tok[rb], k0 + 16 * kb + 4 * q4 + r - P)) s[rb][kb][r] = -INFINITY;
      }
    }
    if constexpr (X == kScores) {
      // (each element by itself: the vector times a.cx became a 16-byte load
      // of the arguments at cx, and that a copy of them per lane, in LDS;
      // 22 us against 8.5 on a step of one sequence)
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r) scored[rb][kb][r] = s[rb][kb][r] * a.cx;
    }
    float corr[NRB];
    typename E::v8 pf[NRB];
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
      float mx = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[rb][kb][r]);
      mx = xor32_max(xor16_max(mx));
      const float m_new = fmaxf(m_run[rb], mx * a.cx);
      corr[rb] = fast_exp2(m_run[rb] - m_new);
      m_run[rb] = m_new;
      float rs = 0.f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = fast_exp2(fmaf(s[rb][kb][r], a.cx, -m_new));
          rs += p;
          s[rb][kb][r] = p;
        }
      l_run[rb] = fmaf(l_run[rb], corr[rb], rs);
      // The weights enter their product with V rounded to the 16-bit type, as the flash
      // forward's do (the matrix instruction takes both operands in it; at most half a
      // step of sum p |v|); their sum takes them unrounded.
      // P^T as the B operand: slot j < 4 <-> key 4*q4 + j, slot j >= 4 <-> key 16 + 4*q4 + j - 4.
      u32x4 pk;
      pk[0] = E::pack2(s[rb][0][0], s[rb][0][1]);
      pk[1] = E::pack2(s[rb][0][2], s[rb][0][3]);
      pk[2] = E::pack2(s[rb][1][0], s[rb][1][1]);
      pk[3] = E::pack2(s[rb][1][2], s[rb][1][3]);
      pf[rb] = E::as8(pk);
    }
    wave_lds_sync();
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
      const u32x2 lo = *(const u32x2*)(vl + vt_at(16 * db + c16, q4));
      const u32x2 hi = *(const u32x2*)(vl + vt_at(16 * db + c16, q4 + 4));
      const u32x4 av = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb) {
        acc[rb][db] *= corr[rb];
        acc[rb][db] = E::mma16(E::as8(av), pf[rb], acc[rb][db]);
      }
    }
    wave_lds_sync();
    if constexpr (X == kTree) {
      if (unbounded)
        add_unbounded<NRB, NDB>(a, tree, tree_p + 512 * w, s, acc, tok, k0, w1, P, [&](int key, int db, int& odd) {
          const int d = 16 * db + 4 * q4;
          if (ROWS && d >= rdv) return f32x4{};
          const u32x2 u = *(const u32x2*)(Vb + (size_t)key * v_tok + d);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t diff = u[e] ^ finite_halves<E>(u[e]);
            odd |= ((diff & 0xffffu) ? 1 << 2 * e : 0) | ((diff >> 16) ? 2 << 2 * e : 0);
          }
          return f32x4{E::lo(u[0]), E::hi(u[0]), E::lo(u[1]), E::hi(u[1])};
        });
    }
  }

  if constexpr (X == kScores)
    if (w0 < w1) store_scores((w1 - w0 - 1) / 32 * 32 + w0);

  // ---- combine the 4 waves of this work item, one row block at a time ----
  const bool final_out = c0 == 0 && L <= a.chunk;
  const size_t part = (size_t)bg * a.nch + chunk_id;
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb)
    combine_rows<DV, X>(a, (float*)vt_lds, acc[rb], [&](int i) { return 4 * i + q4; }, has[rb] ? m_run[rb] : kMaxInit,
                        has[rb] ? xor32_sum(xor16_sum(l_run[rb])) : 0.f, row0, rb, b, g, part, final_out);
}

// ---------------------------------------------------------------------------
// fp32 GQA split-KV decode: the work items and wave split of
// gqa_decode_kernel with full fp32 products on v_mfma_f32_16x16x4f32
// (A lane l holds A[l%16][l/16], B lane l holds B[l/16][l%16], C as
// 16x16x32).  Q.K contracts dims d = 16j + 4*q4 + e in step (j, e) with k
// index q4, so each lane's K and Q^T operands are float4 loads of dims
// 16j + 4*q4 .. +3.  P.V's B operand for step e is the score register e
// itself (keys 4*q4 + e of a 16-key block), and its A operand V[key][dim] is
// loaded per lane, 4 consecutive dims, one for each of 4 blocks (block i's rows are
// the dims 64(i/4) + 4*row + i%4).  Up to 32 rows (2 row blocks).
// ---------------------------------------------------------------------------
__device__ __forceinline__ f32x4 mfma16x16x4f32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

template <int D, int DV, int NRB, int X>
__device__ __forceinline__ void gqa_decode_f32(const DecodeArgs& a) {
  constexpr int NJ = D / 16;    // float4 groups of Q.K per lane
  constexpr int NDB = DV / 16;  // 16-dim output blocks
  static_assert(D % 64 == 0 && DV % 64 == 0 && NRB <= 2, "fp32 decode shape");
  __shared__ __attribute__((aligned(16))) float red[4 * 16 * DV + 4 * 16 * 2];

  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int c16 = lane & 15, q4 = lane >> 4;
  __shared__ int sched[4 + 2 * kSchedMaxBatch];
  int b, g, chunk_id, L;
  if (!decode_item(a, sched, b, g, chunk_id, L, blockIdx.x)) return;
  const int bg = b * a.G + g;
  const int c0 = chunk_id * a.chunk;
  const int per_wave = ((min(L - c0, a.chunk) + 127) >> 7) << 5;
  const int w0 = c0 + w * per_wave;
  const int w1 = min(w0 + per_wave, L);
  const float* Q = (const float*)a.q;
  const size_t k_tok = X == kPlain ? (size_t)a.G * D : (size_t)a.k_t;
  const size_t v_tok = X == kPlain ? (size_t)a.G * DV : (size_t)a.v_t;
  const float* Kb =
      (const float*)a.k + (X == kPlain ? ((size_t)b * a.Lk * a.G + g) * D : (size_t)(b * a.k_b + g * a.k_h));
  const float* Vb =
      (const float*)a.v + (X == kPlain ? ((size_t)b * a.Lk * a.G + g) * DV : (size_t)(b * a.v_b + g * a.v_h));
  const int row0 = blockIdx.y * 16 * NRB;  // this row group's first row
  const int P = X == kTree ? prefix_len(a, b) : 0;
  __shared__ typename std::conditional<X == kTree, TreeTable, int>::type tree;
  __shared__ float tree_p[X == kTree ? 4 * 512 : 1];
  if constexpr (X == kTree) {
    if (c0 + a.chunk > P) build_tree<kDecThreads / 64>(a, b, tree);
  }
  int tok[NRB];
  bool has[NRB];

  f32x4 qf[NRB][NJ];
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb) {
    const int row = row0 + 16 * rb + c16;
    const bool rv = row < a.rows;
    int t = 0, h = 0;
    if (rv) row_to_head(a, g, row, t, h);
    tok[rb] = t;
    has[rb] = X != kTree || tree_token(a, b, t);
    const float* qrow = Q + ((size_t)(b * a.Lq + t) * a.Hq + h) * D;
#pragma unroll
    for (int j = 0; j < NJ; ++j) qf[rb][j] = rv ? *(const f32x4*)(qrow + 16 * j + 4 * q4) : f32x4{};
  }
  f32x4 acc[NRB][NDB];
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb)
#pragma unroll
    for (int i = 0; i < NDB; ++i) acc[rb][i] = f32x4{};
  float m_run[NRB], l_run[NRB];
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb) {
    m_run[rb] = kMaxInit;
    l_run[rb] = 0.f;
  }

  for (int k0 = w0; k0 < w1; k0 += 32) {
    // (loads without a condition, all issued before the first is used)
    f32x4 kf[2][NJ];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      const float* kp = Kb + (size_t)min(k0 + 16 * kb + c16, w1 - 1) * k_tok + 4 * q4;
#pragma unroll
      for (int j = 0; j < NJ; ++j) kf[kb][j] = *(const f32x4*)(kp + 16 * j);
    }
    // V[key 16kb + 4*q4 + e][dim 64(i/4) + 4*c16 + i%4] for the A operands of P.V, as
    // bits: 16 bytes a load, which give the rows of four blocks (a dword a load, of
    // dims 16i + c16: 5 us of 17 to issue, at 128 dims)
    uint32_t vv[2][4][NDB];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = k0 + 16 * kb + 4 * q4 + e;
        const float* vp = Vb + (size_t)min(key, w1 - 1) * v_tok + 4 * c16;
#pragma unroll
        for (int i = 0; i < NDB; i += 4) {
          const u32x4 u = *(const u32x4*)(vp + 16 * i);
#pragma unroll
          for (int t = 0; t < 4; ++t) vv[kb][e][i + t] = u[t];
        }
      }
    // S^T for keys k0 + 16*kb + 4*q4 + r, query row 16rb + c16.
    f32x4 s[NRB][2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb) {
        s[rb][kb] = f32x4{};
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[rb][kb] = mfma16x16x4f32(kf[kb][j][e], qf[rb][j][e], s[rb][kb]);
      }
    }
    if (k0 + 32 > w1) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < NDB; ++i) vv[kb][e][i] = k0 + 16 * kb + 4 * q4 + e < w1 ? vv[kb][e][i] : 0u;
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (k0 + 16 * kb + 4 * q4 + r >= w1) s[rb][kb][r] = -INFINITY;
    }
    bool unbounded = false;  // as in gqa_decode
    if constexpr (X == kTree) {
      if (k0 + 32 > P) {
        bool any = false;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int i = 0; i < NDB; ++i) {
              const bool out = not_finite(vv[kb][e][i]);
              any |= out;
              vv[kb][e][i] = out ? 0u : vv[kb][e][i];
            }
#pragma unroll
            for (int rb = 0; rb < NRB; ++rb)
              if (!tree_sees(tree, a.Lq, tok[rb], k0 + 16 * kb + 4 * q4 + e - P)) s[rb][kb][e] = -INFINITY;
          }
        unbounded = wave_any(any);
      }
    }
    if constexpr (X == kScores) {
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb) {
        const int row = row0 + 16 * rb + c16;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const int key = k0 + 16 * kb + 4 * q4;
          // (each element by itself: the vector times a.cx became a 16-byte load
          // of the arguments at cx, and that a copy of them per lane, in LDS;
          // 22 us against 8.5 on a step of one sequence)
          f32x4 x;
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] = s[rb][kb][r] * a.cx;
          if (row < a.rows && key < w1) *(f32x4*)(a.scores + ((size_t)bg * a.rows + row) * a.score_ld + key) = x;
        }
      }
    }
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
      float mx = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[rb][kb][r]);
      mx = xor32_max(xor16_max(mx));
      const float m_new = fmaxf(m_run[rb], mx * a.cx);
      const float corr = fast_exp2(m_run[rb] - m_new);
      m_run[rb] = m_new;
      float rs = 0.f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = fast_exp2(fmaf(s[rb][kb][r], a.cx, -m_new));
          rs += p;
          s[rb][kb][r] = p;
        }
      l_run[rb] = fmaf(l_run[rb], corr, rs);
#pragma unroll
      for (int i = 0; i < NDB; ++i) {
        acc[rb][i] *= corr;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[rb][i] = mfma16x16x4f32(__uint_as_float(vv[kb][e][i]), s[rb][kb][e], acc[rb][i]);
      }
    }
    if constexpr (X == kTree) {
      if (unbounded)
        add_unbounded<NRB, NDB>(a, tree, tree_p + 512 * w, s, acc, tok, k0, w1, P, [&](int key, int db, int& odd) {
          const uint32_t* vr = (const uint32_t*)(Vb + (size_t)key * v_tok) + 64 * (db / 4) + 16 * q4 + db % 4;
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t u = vr[4 * e];
            odd |= not_finite(u) ? 1 << e : 0;
            v[e] = __uint_as_float(u);
          }
          return v;
        });
    }
  }

  const bool final_out = c0 == 0 && L <= a.chunk;
  const size_t part = (size_t)bg * a.nch + chunk_id;
#pragma unroll
  for (int rb = 0; rb < NRB; ++rb) {
    f32x4 o[NDB];  // quad 16j + 4*q4 + r: element r of the four blocks 4j ..
#pragma unroll
    for (int i = 0; i < NDB; ++i)
#pragma unroll
      for (int t = 0; t < 4; ++t) o[i][t] = acc[rb][i / 4 * 4 + t][i % 4];
    combine_rows<DV, X>(a, red, o, [&](int i) { return i / 4 * 16 + 4 * q4 + i % 4; }, has[rb] ? m_run[rb] : kMaxInit,
                        has[rb] ? xor32_sum(xor16_sum(l_run[rb])) : 0.f, row0, rb, b, g, part, final_out);
  }
}

// Exact merge of the chunk partials of one (batch, group, query row):
// M = max_c m_c, O = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c
// (attention_splitkv.py:236-245, with unnormalised partials).  One thread per
// 4 output dims.  The partials are taken in batches of kMergeBatch chunks whose
// loads (m, l and 4 dims of O per chunk) are all issued before any is used, so
// a batch costs one memory round trip (the first one overlapping the length
// load); batches are combined online (running max, rescaled sums).  Sequences that fit one chunk were finished by the
// chunk kernel; empty sequences (length 0, no chunk ran) get a zero output and
// LSE = +inf (attention_xla.py:417-420).
constexpr int kMergeThreads = 128;
constexpr int kMergeBatch = 16;
template <int BATCH = kMergeBatch>
__device__ __forceinline__ void merge_chunks(const DecodeArgs& a, long gid) {
  const int nq = a.orow / 4;
  const long item = gid / nq;
  const int u = (int)(gid % nq);
  if (item >= (long)a.B * a.G * a.rows) return;
  const int bg = (int)(item / a.rows), r = (int)(item % a.rows);
  const int b = bg / a.G, g = bg % a.G;
  const size_t base = (size_t)bg * a.nch;
  const float* ml = a.ws_ml + (base * a.rows + r) * 2;  // chunk c at ml[c * ml_stride]
  const size_t ml_stride = (size_t)a.rows * 2;
  const float* po = a.ws_o + (base * a.rows + r) * a.dv + 4 * u;  // chunk c at po[c * o_stride]
  const size_t o_stride = (size_t)a.rows * a.dv;
  // The sequence length is needed only after the first batch's loads are
  // issued: partial addresses are clamped to the workspace's a.nch chunks,
  // and slots at or past this sequence's chunk count n (never written by this
  // call) are dropped by selects, so whatever they hold cannot leak in.
  // (A buffer load of the length: unconditional, so nothing waits for it
  // before the partial loads; without lengths the buffer is empty.)
  const int len_raw = (int)__builtin_amdgcn_raw_buffer_load_b32(
      make_rsrc(a.lengths, a.lengths ? (uint32_t)a.B * 4u : 0u), b * 4, 0, 0);
  float M = kMaxInit, den = 0.f;
  f32x4 num = {0.f, 0.f, 0.f, 0.f};
  float mv[BATCH], lv[BATCH];
  f32x4 ov[BATCH];
  auto load_batch = [&](int c0) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const size_t c = (size_t)min(c0 + i, a.nch - 1);
      mv[i] = ml[c * ml_stride];
      lv[i] = ml[c * ml_stride + 1];
      ov[i] = *(const f32x4*)(po + c * o_stride);
    }
    __builtin_amdgcn_sched_barrier(0);  // keep every load of the batch ahead of the arithmetic
  };
  auto add_batch = [&](int c0, int n) {
    float bm = M;
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (c0 + i < n) bm = fmaxf(bm, mv[i]);
    const float sc = fast_exp2(M - bm);
    M = bm;
    den *= sc;
    num *= sc;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (c0 + i < n) {
        const float wt = fast_exp2(mv[i] - M);
        den = fmaf(wt, lv[i], den);
        num += wt * ov[i];
      }
    }
  };
  load_batch(0);
  const int L = a.lengths ? min(a.Lk, min(a.Lk, max(len_raw, 0)) + a.extra) : a.Lk;  // as seq_len
  const int n = (L + a.chunk - 1) / a.chunk;
  if (n == 1) return;  // the chunk kernel wrote this row's output
  add_batch(0, n);
  for (int c0 = BATCH; c0 < n; c0 += BATCH) {
    load_batch(c0);
    add_batch(c0, n);
  }
  int t, h;
  row_to_head(a, g, r, t, h);
  const bool some = a.extra ? some_key(den) : den > 0.f;
  const float inv = some ? 1.f / den : 0.f;
  const size_t oi = ((size_t)(b * a.Lq + t) * a.Hq + h) * a.orow + 4 * u;
  if (a.o32) {
    *(f32x4*)(a.o32 + oi) = num * inv;
  } else {
    const u32x2 pk = a.f16 ? u32x2{F16Fmt::pack2(num[0] * inv, num[1] * inv), F16Fmt::pack2(num[2] * inv, num[3] * inv)}
                           : u32x2{Bf16Fmt::pack2(num[0] * inv, num[1] * inv), Bf16Fmt::pack2(num[2] * inv, num[3] * inv)};
    *(u32x2*)(a.o + oi) = pk;
  }
  if (a.lse && u == 0)
    a.lse[((size_t)b * a.Hq + h) * a.Lq + t] = some ? (M + __log2f(den)) * kLn2 : INFINITY;
}

// ---------------------------------------------------------------------------
// Host (decode.hip)
// ---------------------------------------------------------------------------
constexpr int64_t kGqaItems = 1024;  // work items an automatic chunk leaves at most (auto_chunk)
constexpr int64_t kMlaItems = 256;
constexpr int64_t kStreamBytes = (int64_t)768 << 20;  // cache bytes past which it is streamed (decode_streams_kv)
int64_t auto_chunk(int64_t batch, int64_t groups, int64_t kv_len, int64_t items);
size_t ws_size(int64_t batch, int64_t groups, int64_t rows, int64_t kv_len, int64_t v_dim, int64_t chunk);
bool decode_streams_kv(int64_t cache_bytes, int64_t threshold);
int gqa_row_blocks(int64_t rows, int64_t head_dim, int64_t v_dim, bool f32);
// Checks the arguments of a decode of the cache operators (tree_decode.hip,
// key_weights.hip), resolves chunk = 0 and fills `a`; a PJX_* status.
int fill_cache_decode(DecodeArgs& a, const char* who, int dtype, const void* q, const void* k, const void* v,
                      const int32_t* kv_lengths, void* o, float* lse, int64_t batch, int64_t q_len, int64_t kv_len,
                      int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t row_dim,
                      const pjx_cache_strides* strides, float sm_scale, int64_t chunk);
// Drafts of many rows (tree_wide.hip): whether its kernel takes them, and the
// launch (auto_chunk_size: the chunk is the kernel's to choose, from a.chunk up).
bool tree_wide_takes(const DecodeArgs& a, int head_dim, bool f32);
int run_tree_wide(DecodeArgs& a, int head_dim, bool auto_chunk_size, void* ws, size_t ws_bytes, hipStream_t s,
                  const char* who);
// Merges the chunk partials of a decode whose chunk kernel was launched with `a`.
int launch_decode_merge(const DecodeArgs& a, hipStream_t stream, const char* name);
// The same where a row has at most kFewChunks partials.
constexpr int kFewChunks = 4;
int launch_merge_few(const DecodeArgs& a, hipStream_t stream, const char* name);

// Launches chunk kernel K over the work items of `a`, whose partials it places
// in the workspace.
template <auto K>
int run_chunks(DecodeArgs& a, void* workspace, size_t ws_bytes, hipStream_t stream, const char* name) {
  if (a.orow == 0) a.orow = a.dv;
  const size_t need = ws_size(a.B, a.G, a.rows, a.Lk, a.dv, a.chunk);
  if (!workspace || ws_bytes < need) return fail(PJX_ERR_WORKSPACE, "decode: workspace missing or too small");
  const size_t parts = (size_t)a.B * a.G * a.nch * a.rows;
  a.ws_o = (float*)workspace;
  a.ws_ml = a.ws_o + parts * a.dv;
  const long blocks = (long)a.B * a.G * a.nch;
  const long groups = ((long)a.rows + a.rpg - 1) / a.rpg;
  if (blocks > 0x7fffffffL || groups > 65535 || (long)a.B * a.G * a.rows > 0x7fffffffL)
    return fail(PJX_ERR_INVALID, "decode: grid too large");
  launch_kernel<K>(dim3((unsigned)blocks, (unsigned)groups), dim3(kDecThreads), 0, stream, a);
  return check_launch(name);
}

template <auto K>
int run_decode(DecodeArgs& a, void* workspace, size_t ws_bytes, hipStream_t stream, const char* name) {
  const int rc = run_chunks<K>(a, workspace, ws_bytes, stream, name);
  // (a draft has a key at least, so one chunk's kernel wrote every row)
  if (rc || (a.extra && a.nch == 1)) return rc;
  return a.extra && a.nch <= kFewChunks ? launch_merge_few(a, stream, name) : launch_decode_merge(a, stream, name);
}

}  // namespace pjx
