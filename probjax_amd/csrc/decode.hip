// Split-KV decode for gfx950: GQA decode (separate K/V, per-sequence lengths)
// and absorbed latent attention (MLA, K = V = one shared latent cache).
//
// Semantics: the split-KV forward of probjax
// (probjax/nn/pallas_kernels/kernels/attention_splitkv.py:43-250) -- every
// KV chunk yields a partial output and its softmax statistics, combined by an
// exact log-sum-exp merge -- extended with KVLenMask (keys >= L[b] masked,
// attention_mask_bias.py:1399-1532), whose reference semantics are those of
// xla_attention (kernels/attention_xla.py:339-429).  Query rows are packed per
// KV head: row = g*Lq + t for GQA (attention_splitkv.py:121-126) and
// row = t*H + h for MLA (heads folded, layers/latent_attention.py:458-469).
//
// Work decomposition (HBM-bound; compute is a few % of the MFMA rate):
//   * one workgroup per (batch, kv group, chunk of `chunk` keys); chunks past
//     the sequence's length exit at once, so only valid K/V is ever read;
//   * GQA (gqa_decode_kernel): the 4 waves split the chunk's keys, load K rows
//     straight into MFMA operands and V through a per-wave LDS slab, and
//     combine their (max, sum, O) in LDS at the end;
//   * latent (mla_decode_kernel): 64-key tiles of the shared latent go
//     HBM -> LDS; each wave forms S^T for 16 keys, the 64 x 16 score tile is
//     shared through LDS, every wave runs the same online softmax over it and
//     multiplies its own quarter of the output dims, so no combine is needed;
//   * the merge kernel combines the chunks of one (batch, group) exactly.
// Inputs are bf16 or fp16 (the kernels are templated on the 16-bit format;
// the v_mfma_*_bf16 named here are v_mfma_*_f16 for fp16) or fp32 (GQA only).
#include <stdio.h>
#include <stdlib.h>

#include <atomic>

#include "decode_common.h"

namespace pjx {

template <typename E, int D, int DV, int NRB, bool STREAM>
__global__ __launch_bounds__(256, (decode_occupancy<D, DV, NRB>())) void gqa_decode_kernel(DecodeArgs a) {
  gqa_decode<E, D, DV, NRB, STREAM, false>(a);
}

// Head dims that are no kernel width, on the cache as it lies in memory: bound
// by its bytes, like the kernels above, at about the rate of a plain copy.
// Zero-padding the cache to the width on every step read it once and wrote and
// read it width / dim times as large.  bf16, us, padded -> rows (B, S, Hq, Hkv,
// D): (1,2048,8,8,80) 43 -> 14; (16,8192,32,8,96) 388 -> 85; (32,8192,32,8,80)
// 831 -> 153 (4.4 TB/s); (32,8192,32,8,40) 536 -> 129.  Non-temporal loads, which
// need whole 128-byte lines, were slower at every size (1.3 GB at D = 80: 326
// against 294 us), so these rows always take ordinary ones.
template <typename E, int D, int NRB>
__global__ __launch_bounds__(256, (decode_occupancy<D, D, NRB>())) void gqa_decode_rows_kernel(DecodeArgs a) {
  gqa_decode<E, D, D, NRB, false, true>(a);
}

// Two waves per SIMD where 256 registers do: one 16-row block of widths 128 and 256
// needs 262 otherwise (8 sequences of 2048 keys, 4 KV heads: 29.7 us).
template <int D, int DV, int NRB>
__global__ __launch_bounds__(256, NRB == 1 && D + DV < 512 ? 2 : 1) void gqa_decode_f32_kernel(DecodeArgs a) {
  gqa_decode_f32<D, DV, NRB, kPlain>(a);
}

// ---------------------------------------------------------------------------
// Latent (MLA) decode: K = V = one shared latent cache row of D dims per key,
// the first DV dims acting as values.  One workgroup = one (chunk, batch)
// item; the two LDS stages (2 x 64 keys x 2D bytes) leave room for one
// workgroup per CU.
//   * Each 64-key tile is contiguous in HBM (64 rows x 2D bytes) and is copied
//     HBM -> LDS with buffer->LDS loads, 1 KiB per wave instruction; the next
//     tile is in flight while the current one is computed.
//   * Wave w forms S^T = K Q^T for keys [16w, 16w+16) of every tile with
//     v_mfma_f32_16x16x32_bf16 (K rows from LDS, Q^T in registers) and writes
//     it to LDS (1 KiB); after a barrier every wave reads the whole 64 x 16
//     score tile, runs the online softmax over it (the same values in every
//     wave) and computes O^T += V^T P^T for its DV/4 output dims over all 64
//     keys with v_mfma_f32_16x16x16_bf16, whose B operands are the shared
//     score blocks as they stand (the C layout of S^T is the B layout of
//     P^T) and whose A operands (V^T) come from the same LDS tile through
//     ds_read_b64_tr_b16.  The latent row is read from HBM once and from LDS
//     twice.
//   * Each wave ends with the finished (max, sum, O) of its dims: nothing is
//     combined across waves (a combine of four key-split partials through LDS
//     took ~2.6 us of the C5 step).
// LDS rows keep their 16-byte columns XOR-swizzled per row (within aligned
// groups of 8 or 16 columns), so that 16 lanes reading one column of 16 rows
// (K fragments) and 32 lanes reading two columns of 8 rows (transposing V
// reads) touch distinct banks.
// ---------------------------------------------------------------------------
template <int D>
struct LatentTile {
  static constexpr int BK = 64;                    // keys per tile
  static constexpr int ROWB = 2 * D;               // bytes per latent row
  static constexpr int NC = D / 8;                 // 16-byte columns per row
  static constexpr int STAGE_B = BK * ROWB;        // bytes per stage
  static constexpr int NLD = STAGE_B / (4 * 1024);  // 1 KiB loads per wave per tile
  static constexpr int GRP = (NC % 16 == 0) ? 16 : 8;  // swizzle group (columns)
  static_assert(NC % 8 == 0 && STAGE_B % 4096 == 0, "latent tile shape");
  // Row r's column XOR.  Row r starts at 16-byte bank unit (r*NC) % 16, which
  // is 0 when NC % 16 == 0 and 8*(r&1) when NC % 16 == 8.  K fragments
  // (ds_read_b128) have lane l read column 4e + l/16 of row l%16, and gfx950's
  // LDS serves lanes 0-7 with 24-31 and 8-15 with 16-23 in one cycle, so rows
  // r < 8 of column 4e and rows r + 8 of column 4e + 1 must take different
  // bank groups: XOR 2(r&7) (whole lines) or r&6 (half lines) sends the first
  // to even groups and the second to odd ones.  The transposing V^T reads
  // (32 lanes: an aligned column pair of 8 consecutive rows) stay distinct.
  __device__ static int swz(int r) { return GRP == 16 ? ((r & 7) << 1) : (r & 6); }
};

template <typename E, int D, int DV, bool STREAM>
__global__ __launch_bounds__(kDecThreads, 1) void mla_decode_kernel(DecodeArgs a) {
  using T = LatentTile<D>;
  constexpr int BK = T::BK, ROWB = T::ROWB, NLD = T::NLD, GRP = T::GRP;
  constexpr int KSTEPS = D / 32;  // 32-dim k-steps of Q.K
  constexpr int SPG = GRP / 4;    // k-steps per swizzle group
  constexpr int NDT = DV / 16;    // 16-dim output tiles
  constexpr int NDW = NDT / 4;    // output tiles of one wave
  constexpr int DPG = GRP / 2;    // output tiles per swizzle group
  static_assert(DV % 64 == 0 && DV <= D, "value dims are a prefix of the latent row");
  static_assert(KSTEPS % SPG == 0 && NDT % DPG == 0, "swizzle groups");
  __shared__ __attribute__((aligned(1024))) unsigned char smem0[T::STAGE_B];
  __shared__ __attribute__((aligned(1024))) unsigned char smem1[T::STAGE_B];
  __shared__ f32x4 sx[4 * 64];  // the tile's S^T blocks, one per wave, in MFMA C layout

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, q4 = lane >> 4;
  __shared__ int sched[4 + 2 * kSchedMaxBatch];
  int b, g, chunk_id, L;
  if (!decode_item(a, sched, b, g, chunk_id, L, blockIdx.x)) return;  // nothing past the length is read
  const int c0 = chunk_id * a.chunk;
  const int c1 = min(c0 + a.chunk, L);
  const int n_tiles = (c1 - c0 + BK - 1) / BK;

  // Q^T as the B operand: lane holds query row row0 + c16 (16 rows per row
  // group, blockIdx.y), dims 32*s + 8*q4 + [0,8).
  const int row = blockIdx.y * 16 + c16;
  typename E::v8 qf[KSTEPS];
  {
    const bool rv = row < a.rows;
    int t = 0, h = 0;
    if (rv) row_to_head(a, 0, row, t, h);
    const uint16_t* qrow = a.q + ((size_t)(b * a.Lq + t) * a.Hq + h) * D;
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      u32x4 r = {0u, 0u, 0u, 0u};
      if (rv) r = *(const u32x4*)(qrow + 32 * s + 8 * q4);
      qf[s] = E::as8(r);
    }
  }
  const unsigned char* Kb = (const unsigned char*)a.k + (size_t)b * a.Lk * ROWB;

  // Buffer->LDS sources: load j of wave w fills 16-byte LDS unit
  // p = (NLD*w + j)*64 + lane = row*NC + slot with global column slot ^ swz(row).
  uint32_t voff[NLD];
#pragma unroll
  for (int j = 0; j < NLD; ++j) {
    const int p = (NLD * w + j) * 64 + lane, r = p / T::NC, slot = p % T::NC;
    voff[j] = r * ROWB + 16 * (slot ^ T::swz(r));
  }
  // K fragment of k-step s: row 16w + c16, column 4s + q4, i.e. group s / SPG,
  // column 4*(s % SPG) + q4 within it.
  uint32_t offK[SPG];
  {
    const int r = 16 * w + c16;
#pragma unroll
    for (int e = 0; e < SPG; ++e) offK[e] = r * ROWB + 16 * ((4 * e + q4) ^ T::swz(r));
  }
  // Transposing V^T read for output tile dt (dims 16*dt + [0,16)) and key
  // block kb (keys 16kb + 4*q4 + [0,4)): lane s of each 16-lane group points
  // at row 16kb + 4*q4 + s/4, dims 16*dt + 4*(s%4) + [0,4).  The swizzle of a
  // row depends on it modulo 16 only, so key block kb is offV + 16*kb rows.
  uint32_t offV[DPG];
  {
    const int r = 4 * q4 + (c16 >> 2);
#pragma unroll
    for (int e = 0; e < DPG; ++e)
      offV[e] = r * ROWB + 16 * ((2 * e + ((c16 & 3) >> 1)) ^ T::swz(r)) + 8 * (c16 & 1);
  }

  // acc[i] = O^T[dims 16*(NDW*w + i) + 4*q4 + r][row c16]
  f32x4 acc[NDW];
#pragma unroll
  for (int i = 0; i < NDW; ++i) acc[i] = f32x4{};
  float m_run = kMaxInit, l_run = 0.f;

  auto issue = [&](int t, unsigned char* ks) {
    const int k0 = c0 + t * BK;
    // Rows at or past c1 read as 0; a tile past the chunk reads nothing.
    // (readfirstlane: the clamp is computed on the vector unit, and a vector
    // operand of the buffer descriptor would need a waterfall loop.)
    const uint32_t bytes = __builtin_amdgcn_readfirstlane(max(0, min(BK, c1 - k0)) * ROWB);
    const rsrc_t rs = make_rsrc(Kb + (size_t)k0 * ROWB, bytes);
#pragma unroll
    for (int j = 0; j < NLD; ++j) {
      // STREAM: non-temporal loads for caches past the MALL (as in gqa_decode_kernel)
      if constexpr (STREAM) buffer_load_lds16_nt(rs, ks + (NLD * w + j) * 1024, voff[j]);
      else buffer_load_lds16(rs, ks + (NLD * w + j) * 1024, voff[j]);
    }
  };

  // One tile: wave w forms S^T for its 16 keys and shares it; every wave runs
  // the softmax over all 64 keys (the same values in every wave) and
  // multiplies its own NDW output tiles over all 64 keys.
  auto compute = [&](int t, const unsigned char* ks) {
    const int k0 = c0 + t * BK;
    // s[r] = S^T[key k0 + 16w + 4*q4 + r][row c16]
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < KSTEPS; ++st) {
      const typename E::v8 kf = E::as8(*(const u32x4*)(ks + offK[st % SPG] + 16 * GRP * (st / SPG)));
      s = E::mma16(kf, qf[st], s);
    }
    // Keys at or past c1 -> -inf, selected on every tile (a no-op on full
    // ones) so that the score passes through the vector ALU before its LDS
    // store.  Stored straight from the MFMA accumulator, one instruction
    // after the last MFMA, the value written was sometimes not the finished
    // one when other waves shared the SIMD's matrix pipe (ranks <= 256 run
    // 2-7 workgroups per CU): wrong scores for 4 keys of a row, changing from
    // run to run; 32 wait states before the store, or one workgroup per CU,
    // made every result exact.  A vector-ALU read of an MFMA result is
    // covered by the compiler's MFMA hazard waits; the LDS store's data read
    // was not.
    {
      const int lim = c1 - (k0 + 16 * w + 4 * q4);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] = r < lim ? s[r] : -INFINITY;
    }
    sx[w * 64 + lane] = s;
    stage_barrier();
    f32x4 sk[4];  // sk[kb][r] = S^T[key k0 + 16kb + 4*q4 + r][row c16]
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) sk[kb] = sx[kb * 64 + lane];
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) mx = fmaxf(mx, fmaxf(fmaxf(sk[kb][0], sk[kb][1]), fmaxf(sk[kb][2], sk[kb][3])));
    mx = xor16_max(mx);
    const float mc = xor32_max(mx) * a.cx;
    if (wave_any(mc > m_run + kRescaleLog2)) {
      const float m_new = fmaxf(m_run, mc);
      const float corr = fast_exp2(m_run - m_new);
      m_run = m_new;
      l_run *= corr;
#pragma unroll
      for (int i = 0; i < NDW; ++i) acc[i] *= corr;
    }
    s16x4 pb[4];
    float ls = 0.f;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) p[r] = fast_exp2(fmaf(sk[kb][r], a.cx, -m_run));
      ls += (p[0] + p[1]) + (p[2] + p[3]);
      const u32x2 pk = {E::pack2(p[0], p[1]), E::pack2(p[2], p[3])};
      pb[kb] = __builtin_bit_cast(s16x4, pk);
    }
    l_run += ls;
#pragma unroll
    for (int i = 0; i < NDW; ++i) {
      const int dt = NDW * w + i;
#pragma unroll
      for (int kb = 0; kb < 4; ++kb) {
        const u32x2 av = lds_read_tr16(ks + 16 * kb * ROWB + offV[dt % DPG] + 16 * GRP * (dt / DPG));
        acc[i] = E::mma16k16(__builtin_bit_cast(s16x4, av), pb[kb], acc[i]);
      }
    }
  };

  // Tile t lives in stage t % 2.  Before computing tile t: this wave's loads
  // of it have landed (vmcnt counts loads in issue order and only tile t+1's
  // may still be pending), then the barrier makes every wave's loads visible
  // (each wave reads V^T rows of all four waves).  After computing it, a
  // barrier lets tile t+2 be loaded into the same stage.
  // Every path issues the same sequence of loads (tiles past the chunk are
  // empty) and the loop has no early exit, so the compiler can tell that at
  // each read of a stage the NLD most recent loads target the other stage,
  // and adds no wait of its own.
  // Prologue: Q's loads are waited for while tile 0 is in flight, so that no
  // load into registers is pending at the loop (the compiler would otherwise
  // wait for every outstanding load, tile 1's included, before entering it).
  __builtin_amdgcn_sched_barrier(0);
  issue(0, smem0);
  wait_vmcnt<NLD>();
  issue(1, smem1);
  for (int t = 0; t < n_tiles; t += 2) {
    wait_vmcnt<NLD>();
    stage_barrier();
    compute(t, smem0);
    stage_barrier();
    issue(t + 2, smem0);
    wait_vmcnt<NLD>();
    stage_barrier();
    if (t + 1 < n_tiles) compute(t + 1, smem1);
    stage_barrier();
    issue(t + 3, smem1);
  }
  wait_vmcnt<0>();  // the trailing (empty) tile loads still write LDS

  // Every wave holds the same (max, sum) and the whole output of its dims:
  // no combine across waves.
  l_run = xor16_sum(l_run);
  l_run = xor32_sum(l_run);
  if (row < a.rows) {
    const size_t part = (size_t)b * a.nch + chunk_id;
    const bool final_out = c0 == 0 && L <= a.chunk;
#pragma unroll
    for (int i = 0; i < NDW; ++i)
      emit_row_quad(a, b, 0, row, 16 * (NDW * w + i) + 4 * q4, part, final_out, m_run, l_run, acc[i]);
  }
}

__global__ __launch_bounds__(kMergeThreads) void decode_merge_kernel(DecodeArgs a) {
  merge_chunks(a, (long)blockIdx.x * kMergeThreads + threadIdx.x);
}

// Keys per work item when the caller passes chunk = 0: the smallest power of
// two in [128, 2048] that leaves at most `items` (chunk, batch, group) work
// items at full capacity.  Longer items amortise the per-item start-up (Q
// fragments, the cross-wave combine, partial writes); the item target keeps
// short batches spread over every CU.  Measured on MI355X (GQA, 32 query
// heads over 8 KV heads, D = 128, ragged lengths): ~1024 items at capacity is
// best or within 1% of best for 32 x 8192, 64 x 4096 and full-length 32 x
// 8192 (2048-key chunks) and for 4 x 32768 (1024-key chunks; 2048-key chunks
// leave too few items and take 1.75x as long); the latent decode is fastest
// with ~256 (256-key chunks for 16 x 4096).
int64_t auto_chunk(int64_t batch, int64_t groups, int64_t kv_len, int64_t items) {
  const int64_t work = batch * groups * std::max<int64_t>(kv_len, 1);
  int64_t c = 128;
  while (c < 2048 && work / c > items) c *= 2;
  return c;
}

size_t ws_size(int64_t batch, int64_t groups, int64_t rows, int64_t kv_len,
                      int64_t v_dim, int64_t chunk) {
  // chunk = 0: size for the smaller of the two automatic choices, which is
  // enough for either decode entry point.
  if (chunk <= 0)
    chunk = std::min(auto_chunk(batch, groups, kv_len, kGqaItems), auto_chunk(batch, groups, kv_len, kMlaItems));
  const int64_t nch = (kv_len + chunk - 1) / chunk;
  const int64_t parts = batch * groups * std::max<int64_t>(nch, 1) * rows;
  return (size_t)(parts * v_dim + parts * 2) * sizeof(float);
}

// At most kFewChunks partials a row (wide drafts, tree_wide.hip): the merge above
// issues the loads of 16 whatever there is (8192 rows of 128, 4 chunks: 8 us for 5).
__global__ __launch_bounds__(kMergeThreads) void decode_merge_few_kernel(DecodeArgs a) {
  merge_chunks<kFewChunks>(a, (long)blockIdx.x * kMergeThreads + threadIdx.x);
}

int launch_merge_few(const DecodeArgs& a, hipStream_t stream, const char* name) {
  const long merge_threads = (long)a.B * a.G * a.rows * (a.orow / 4);
  launch_kernel<decode_merge_few_kernel>(dim3((unsigned)((merge_threads + kMergeThreads - 1) / kMergeThreads)),
                     dim3(kMergeThreads), 0, stream, a);
  return check_launch(name);
}

int launch_decode_merge(const DecodeArgs& a, hipStream_t stream, const char* name) {
  const long merge_threads = (long)a.B * a.G * a.rows * (a.orow / 4);
  launch_kernel<decode_merge_kernel>(dim3((unsigned)((merge_threads + kMergeThreads - 1) / kMergeThreads)),
                     dim3(kMergeThreads), 0, stream, a);
  return check_launch(name);
}

// 16-row MFMA column blocks per row group of a GQA decode launch: up to 4 (64
// rows, the reference's largest packed tile, attention_splitkv.py:155-170) at
// head dims <= 128 in bf16 / fp16, else 2; more rows run as several row groups.
int gqa_row_blocks(int64_t rows, int64_t head_dim, int64_t v_dim, bool f32) {
  const int64_t max_nrb = (f32 || head_dim > 128 || v_dim > 128) ? 2 : 4;
  const int64_t need = std::min<int64_t>((rows + kRows - 1) / kRows, max_nrb);
  return need <= 1 ? 1 : need <= 2 ? 2 : 4;
}

// One (D, DV) pair of the 16-bit GQA decode with nrb 16-row blocks per row group.
template <typename E, int D, int DV, bool STREAM>
static int run_gqa_nrb(DecodeArgs& a, int nrb, void* ws, size_t ws_bytes, hipStream_t s, const char* who) {
  if (nrb == 1) return run_decode<gqa_decode_kernel<E, D, DV, 1, STREAM>>(a, ws, ws_bytes, s, who);
  if (nrb == 2) return run_decode<gqa_decode_kernel<E, D, DV, 2, STREAM>>(a, ws, ws_bytes, s, who);
  if constexpr (D <= 128 && DV <= 128) return run_decode<gqa_decode_kernel<E, D, DV, 4, STREAM>>(a, ws, ws_bytes, s, who);
  return fail(PJX_ERR_INVALID, "decode: row blocks");
}

template <typename E, int D, int DV>
static int run_gqa_dims(DecodeArgs& a, int nrb, bool streamed, void* ws, size_t ws_bytes, hipStream_t s,
                        const char* who) {
  return streamed ? run_gqa_nrb<E, D, DV, true>(a, nrb, ws, ws_bytes, s, who)
                  : run_gqa_nrb<E, D, DV, false>(a, nrb, ws, ws_bytes, s, who);
}

// Rows of a.orow <= D elements (gqa_decode_rows_kernel), q/k and v alike.
template <typename E, int D>
static int run_gqa_rows(DecodeArgs& a, int nrb, void* ws, size_t ws_bytes, hipStream_t s, const char* who) {
  if (nrb == 1) return run_decode<gqa_decode_rows_kernel<E, D, 1>>(a, ws, ws_bytes, s, who);
  if (nrb == 2) return run_decode<gqa_decode_rows_kernel<E, D, 2>>(a, ws, ws_bytes, s, who);
  return run_decode<gqa_decode_rows_kernel<E, D, 4>>(a, ws, ws_bytes, s, who);
}

template <typename E>
static int run_gqa_rows_dim(DecodeArgs& a, int head_dim, int nrb, void* ws, size_t ws_bytes, hipStream_t s,
                            const char* who) {
  return head_dim == 64 ? run_gqa_rows<E, 64>(a, nrb, ws, ws_bytes, s, who)
                        : run_gqa_rows<E, 128>(a, nrb, ws, ws_bytes, s, who);
}

template <int D, int DV>
static int run_gqa_f32_dims(DecodeArgs& a, int nrb, void* ws, size_t ws_bytes, hipStream_t s, const char* who) {
  return nrb == 1 ? run_decode<gqa_decode_f32_kernel<D, DV, 1>>(a, ws, ws_bytes, s, who)
                  : run_decode<gqa_decode_f32_kernel<D, DV, 2>>(a, ws, ws_bytes, s, who);
}

// The GQA decode at (head_dim, v_dim), each in {64, 128, 256}: format E (bf16 /
// fp16), or fp32 when F32.
template <typename E, bool F32>
static int run_gqa(DecodeArgs& a, int head_dim, int v_dim, int nrb, bool streamed, void* ws, size_t ws_bytes,
                   hipStream_t s, const char* who) {
#define PJX_GQA_DIMS(D, DV)                                                                   \
  if (head_dim == D && v_dim == DV) {                                                         \
    if constexpr (F32) return run_gqa_f32_dims<D, DV>(a, nrb, ws, ws_bytes, s, who);            \
    else return run_gqa_dims<E, D, DV>(a, nrb, streamed, ws, ws_bytes, s, who);               \
  }
  PJX_GQA_DIMS(64, 64) PJX_GQA_DIMS(64, 128) PJX_GQA_DIMS(64, 256)
  PJX_GQA_DIMS(128, 64) PJX_GQA_DIMS(128, 128) PJX_GQA_DIMS(128, 256)
  PJX_GQA_DIMS(256, 64) PJX_GQA_DIMS(256, 128) PJX_GQA_DIMS(256, 256)
#undef PJX_GQA_DIMS
  return fail(PJX_ERR_INVALID, "decode: head_dim and v_dim must be 64, 128 or 256");
}

// The latent decode (format E) at one (rank, v_dim); STREAM instances when
// `streamed`.
template <typename E, bool STREAM>
static int run_mla_rank(DecodeArgs& a, int64_t rank, int64_t v_dim, void* ws, size_t ws_bytes, hipStream_t s) {
  const char* who = "pjx_mla_decode";
  if (rank == 576 && v_dim == 512) return run_decode<mla_decode_kernel<E, 576, 512, STREAM>>(a, ws, ws_bytes, s, who);
  if (rank == 576 && v_dim == 576) return run_decode<mla_decode_kernel<E, 576, 576, STREAM>>(a, ws, ws_bytes, s, who);
  if (rank == 512 && v_dim == 512) return run_decode<mla_decode_kernel<E, 512, 512, STREAM>>(a, ws, ws_bytes, s, who);
  if (rank == 256 && v_dim == 256) return run_decode<mla_decode_kernel<E, 256, 256, STREAM>>(a, ws, ws_bytes, s, who);
  if (rank == 128 && v_dim == 128) return run_decode<mla_decode_kernel<E, 128, 128, STREAM>>(a, ws, ws_bytes, s, who);
  if (rank == 64 && v_dim == 64) return run_decode<mla_decode_kernel<E, 64, 64, STREAM>>(a, ws, ws_bytes, s, who);
  return fail(PJX_ERR_INVALID,
              "pjx_mla_decode: supported (rank, v_dim): (576,512), (576,576), (512,512), (256,256), (128,128), (64,64)");
}

template <typename E>
static int run_mla_h16(DecodeArgs& a, int64_t rank, int64_t v_dim, bool streamed, void* ws, size_t ws_bytes,
                       hipStream_t s) {
  return streamed ? run_mla_rank<E, true>(a, rank, v_dim, ws, ws_bytes, s)
                  : run_mla_rank<E, false>(a, rank, v_dim, ws, ws_bytes, s);
}

// Whether the 16-bit GQA and latent decodes stream the cache with
// non-temporal loads (the STREAM kernels).  Ordinary loads leave the cache in the 256 MB MALL, which
// repeated calls over a cache that (nearly) fits then hit: measured +3% to
// +17% for STREAM at 537 MB of capacity (~290 MB valid); past that, STREAM
// reads faster (-4% to -9% at 1 GB and more).  The lengths stay on the device,
// so the rule uses the capacity: STREAM above kStreamBytes (3x the MALL).
// The latent decode reads every cached row whole (no ragged tail in the
// measured cases) and crosses over earlier: STREAM measured +1% at 302 MB and
// -10% at 604 MB of latent (R = 576), so its threshold is kStreamBytesLatent.
// PJX_DECODE_STREAM=0 / =1 in the environment forces either kernel.
constexpr int64_t kStreamBytesLatent = (int64_t)512 << 20;
bool decode_streams_kv(int64_t cache_bytes, int64_t threshold) {
  const char* env = getenv("PJX_DECODE_STREAM");
  if (env && env[0] == '0' && env[1] == '\0') return false;
  if (env && env[0] == '1' && env[1] == '\0') return true;
  return cache_bytes > threshold;
}

// Argument checks shared by pjx_splitkv_decode and pjx_splitkv_decode_static
// (everything but the pointers and the workspace); resolves chunk = 0.
static int check_gqa_decode(const char* who, int dtype, int64_t batch, int64_t q_len, int64_t kv_len,
                            int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t v_dim,
                            float sm_scale, int64_t* chunk) {
  char buf[256];
  auto bad = [&](const char* what) {
    snprintf(buf, sizeof(buf), "%s: %s", who, what);
    return fail(PJX_ERR_INVALID, buf);
  };
  if (dtype != PJX_DTYPE_BF16 && dtype != PJX_DTYPE_F16 && dtype != PJX_DTYPE_F32)
    return bad("dtype must be PJX_DTYPE_BF16, PJX_DTYPE_F16 or PJX_DTYPE_F32");
  if (batch < 0 || q_len <= 0 || kv_len < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads)
    return bad("bad sizes");
  auto width = [](int64_t d) { return d == 64 || d == 128 || d == 256; };
  if (!width(head_dim) || !width(v_dim)) return bad("head_dim and v_dim must be 64, 128 or 256");
  if (!(sm_scale > 0.f)) return bad("sm_scale must be > 0");
  if (*chunk == 0) *chunk = auto_chunk(batch, kv_heads, kv_len, kGqaItems);
  if (*chunk < 128 || *chunk % 128) return bad("chunk must be a positive multiple of 128");
  const int64_t rows = (q_heads / kv_heads) * q_len;
  if (kv_len > (1 << 30) || batch * kv_len * kv_heads * std::max(head_dim, v_dim) > ((int64_t)1 << 40) ||
      rows > (1 << 20) || batch * q_heads * q_len * std::max(head_dim, v_dim) > ((int64_t)1 << 40))
    return bad("sizes out of range");
  return PJX_OK;
}

}  // namespace pjx

using namespace pjx;

extern "C" size_t pjx_decode_workspace_size(int64_t batch, int64_t groups, int64_t rows,
                                            int64_t kv_len, int64_t v_dim, int64_t chunk) {
  return ws_size(batch, groups, rows, kv_len, v_dim, chunk);
}

// row_dim: elements of the q, k, v and o rows of a call at head_dim = v_dim, the
// kernel's width (0: rows of head_dim and v_dim).
static int gqa_decode_entry(const char* who, int dtype, const void* q, const void* k, const void* v,
                            const int32_t* kv_lengths, void* o, float* lse, void* workspace,
                            size_t workspace_bytes, int64_t batch, int64_t q_len, int64_t kv_len, int64_t q_heads,
                            int64_t kv_heads, int64_t head_dim, int64_t v_dim, int64_t row_dim, float sm_scale,
                            int64_t chunk, void* stream) {
  clear_error();
  const int vrc = check_gqa_decode(who, dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim, v_dim, sm_scale,
                                   &chunk);
  if (vrc != PJX_OK) return vrc;
  // an empty cache (kv_len == 0) may come as null pointers
  if (!q || !o || (batch * kv_len > 0 && (!k || !v))) {
    char buf[64];
    snprintf(buf, sizeof(buf), "%s: null pointer", who);
    return fail(PJX_ERR_INVALID, buf);
  }
  const bool f32 = dtype == PJX_DTYPE_F32;
  if (batch == 0) return PJX_OK;
  if (kv_len == 0)
    return write_keyless(o, lse, (size_t)(batch * q_len * q_heads * (row_dim ? row_dim : v_dim)), f32, (size_t)(batch * q_heads * q_len),
                         (hipStream_t)stream, who);
  const int64_t rows = (q_heads / kv_heads) * q_len;
  DecodeArgs a = {};
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)k; a.v = (const uint16_t*)v;
  a.lengths = kv_lengths; a.lse = lse;
  if (f32)
    a.o32 = (float*)o;
  else
    a.o = (uint16_t*)o;
  a.f16 = dtype == PJX_DTYPE_F16;
  a.B = (int)batch; a.Lq = (int)q_len; a.Lk = (int)kv_len; a.Hq = (int)q_heads; a.G = (int)kv_heads;
  a.rows = (int)rows; a.fold = 0; a.chunk = (int)chunk;
  a.nch = (int)std::max<int64_t>((kv_len + chunk - 1) / chunk, 1);
  a.dv = (int)v_dim; a.orow = (int)row_dim; a.cx = sm_scale * kLog2e;
  const int nrb = gqa_row_blocks(rows, head_dim, v_dim, f32);
  a.rpg = kRows * nrb;
  hipStream_t s = (hipStream_t)stream;
  const int d = (int)head_dim, dv = (int)v_dim;
  if (row_dim)
    return a.f16 ? run_gqa_rows_dim<F16Fmt>(a, d, nrb, workspace, workspace_bytes, s, who)
                 : run_gqa_rows_dim<Bf16Fmt>(a, d, nrb, workspace, workspace_bytes, s, who);
  const bool streamed = !f32 && decode_streams_kv(batch * kv_len * kv_heads * (head_dim + v_dim) * 2, kStreamBytes);
  if (f32) return run_gqa<Bf16Fmt, true>(a, d, dv, nrb, false, workspace, workspace_bytes, s, who);
  return a.f16 ? run_gqa<F16Fmt, false>(a, d, dv, nrb, streamed, workspace, workspace_bytes, s, who)
               : run_gqa<Bf16Fmt, false>(a, d, dv, nrb, streamed, workspace, workspace_bytes, s, who);
}

extern "C" int pjx_splitkv_decode(int dtype, const void* q, const void* k, const void* v,
                                  const int32_t* kv_lengths, void* o, float* lse,
                                  void* workspace, size_t workspace_bytes, int64_t batch,
                                  int64_t q_len, int64_t kv_len, int64_t q_heads,
                                  int64_t kv_heads, int64_t head_dim, int64_t v_dim, float sm_scale,
                                  int64_t chunk, void* stream) {
  return gqa_decode_entry("pjx_splitkv_decode", dtype, q, k, v, kv_lengths, o, lse, workspace, workspace_bytes, batch,
                          q_len, kv_len, q_heads, kv_heads, head_dim, v_dim, 0, sm_scale, chunk, stream);
}

extern "C" int pjx_splitkv_decode_rows(int dtype, const void* q, const void* k, const void* v,
                                       const int32_t* kv_lengths, void* o, float* lse, void* workspace,
                                       size_t workspace_bytes, int64_t batch, int64_t q_len, int64_t kv_len,
                                       int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t row_dim,
                                       float sm_scale, int64_t chunk, void* stream) {
  clear_error();
  if (dtype != PJX_DTYPE_BF16 && dtype != PJX_DTYPE_F16)
    return fail(PJX_ERR_INVALID, "pjx_splitkv_decode_rows: dtype must be PJX_DTYPE_BF16 or PJX_DTYPE_F16");
  if ((head_dim != 64 && head_dim != 128) || row_dim <= 0 || row_dim % 8 || row_dim > head_dim)
    return fail(PJX_ERR_INVALID,
                "pjx_splitkv_decode_rows: head_dim must be 64 or 128, row_dim a multiple of 8 up to it");
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v) % 16 || (uintptr_t)o % 8)
    return fail(PJX_ERR_INVALID, "pjx_splitkv_decode_rows: q, k, v must start on 16 bytes and o on 8");
  return gqa_decode_entry("pjx_splitkv_decode_rows", dtype, q, k, v, kv_lengths, o, lse, workspace, workspace_bytes,
                          batch, q_len, kv_len, q_heads, kv_heads, head_dim, head_dim, row_dim, sm_scale, chunk,
                          stream);
}

// ---------------------------------------------------------------------------
// Split-KV decode without allocation: the partials live in `scratch`, a
// library-held device array (one copy per GPU, kept until the process ends),
// for callers that cannot allocate (graph capture, serving loops).  Every call
// on a GPU shares that GPU's array: calls that overlap on one GPU race.  No
// part of it needs clearing: the chunk kernel writes every partial the merge
// reads in the same call.
// ---------------------------------------------------------------------------
constexpr size_t kScratchBytes = (size_t)PJX_DECODE_STATIC_SCRATCH_BYTES;
static __device__ __align__(256) unsigned char scratch[kScratchBytes];

constexpr int kMaxDevices = 64;
static std::atomic<void*> g_scratch_ptr[kMaxDevices];

// Device address of the current device's `scratch` (the name itself is only a
// host-side stand-in), looked up on the first call on each device.
static int scratch_ptr(void** out, const char* who) {
  char buf[256];
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess || dev < 0 || dev >= kMaxDevices) {
    snprintf(buf, sizeof(buf), "%s: no usable current device (%s)", who, hipGetErrorString(e));
    return fail(PJX_ERR_LAUNCH, buf);
  }
  void* p = g_scratch_ptr[dev].load(std::memory_order_acquire);
  if (!p) {
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (e != hipSuccess || !p) {
      snprintf(buf, sizeof(buf), "%s: hipGetSymbolAddress(scratch) failed: %s", who, hipGetErrorString(e));
      return fail(PJX_ERR_LAUNCH, buf);
    }
    g_scratch_ptr[dev].store(p, std::memory_order_release);
  }
  *out = p;
  return PJX_OK;
}

extern "C" int pjx_splitkv_decode_static(int dtype, const void* q, const void* k, const void* v,
                                         const int32_t* kv_lengths, void* o, float* lse,
                                         int64_t batch, int64_t q_len, int64_t kv_len,
                                         int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                                         int64_t v_dim, float sm_scale, int64_t chunk, void* stream) {
  clear_error();
  const char* who = "pjx_splitkv_decode_static";
  // every argument check of pjx_splitkv_decode first, then the size of the partials
  const int vrc = check_gqa_decode(who, dtype, batch, q_len, kv_len, q_heads, kv_heads, head_dim, v_dim, sm_scale,
                                   &chunk);
  if (vrc != PJX_OK) return vrc;
  if (batch == 0) return PJX_OK;
  const size_t need = ws_size(batch, kv_heads, (q_heads / kv_heads) * q_len, kv_len, v_dim, chunk);
  if (need > kScratchBytes) {
    char buf[256];
    snprintf(buf, sizeof(buf), "%s: these sizes need %zu bytes of partials, more than the %zu-byte "
             "scratch the library holds; call pjx_splitkv_decode with a workspace", who, need, kScratchBytes);
    return fail(PJX_ERR_WORKSPACE, buf);
  }
  void* ws = nullptr;
  const int rc = scratch_ptr(&ws, who);
  if (rc != PJX_OK) return rc;
  return pjx_splitkv_decode(dtype, q, k, v, kv_lengths, o, lse, ws, kScratchBytes, batch, q_len, kv_len,
                            q_heads, kv_heads, head_dim, v_dim, sm_scale, chunk, stream);
}

extern "C" int pjx_mla_decode(int dtype, const void* q, const void* cache,
                              const int32_t* kv_lengths, void* o, float* lse, void* workspace,
                              size_t workspace_bytes, int64_t batch, int64_t q_len,
                              int64_t heads, int64_t kv_len, int64_t rank, int64_t v_dim,
                              float sm_scale, int64_t chunk, void* stream) {
  clear_error();
  if (dtype != PJX_DTYPE_BF16 && dtype != PJX_DTYPE_F16)
    return fail(PJX_ERR_INVALID, "pjx_mla_decode: dtype must be PJX_DTYPE_BF16 or PJX_DTYPE_F16");
  // an empty cache (kv_len == 0) may come as a null pointer
  if (!q || !o || (batch * kv_len > 0 && !cache)) return fail(PJX_ERR_INVALID, "pjx_mla_decode: null pointer");
  if (batch < 0 || q_len <= 0 || heads <= 0 || kv_len < 0) return fail(PJX_ERR_INVALID, "pjx_mla_decode: bad sizes");
  if (q_len * heads > (1 << 20)) return fail(PJX_ERR_INVALID, "pjx_mla_decode: Lq*H must be <= 2^20");
  if (!(sm_scale > 0.f)) return fail(PJX_ERR_INVALID, "pjx_mla_decode: sm_scale must be > 0");
  if (chunk == 0) chunk = auto_chunk(batch, 1, kv_len, kMlaItems);
  if (chunk < kTile || chunk % kTile) return fail(PJX_ERR_INVALID, "pjx_mla_decode: chunk must be a positive multiple of 64");
  if (kv_len > (1 << 30) || batch * kv_len * rank > ((int64_t)1 << 40))
    return fail(PJX_ERR_INVALID, "pjx_mla_decode: sizes out of range");
  DecodeArgs a = {};
  a.q = (const uint16_t*)q; a.k = (const uint16_t*)cache; a.v = (const uint16_t*)cache;
  a.lengths = kv_lengths; a.o = (uint16_t*)o; a.lse = lse;
  a.B = (int)batch; a.Lq = (int)q_len; a.Lk = (int)kv_len; a.Hq = (int)heads; a.G = 1;
  a.rows = (int)(q_len * heads); a.fold = 1; a.chunk = (int)chunk;
  a.nch = (int)std::max<int64_t>((kv_len + chunk - 1) / chunk, 1);
  a.dv = (int)v_dim; a.cx = sm_scale * kLog2e;
  a.rpg = kRows;  // one 16-row MFMA column block per row group
  hipStream_t s = (hipStream_t)stream;
  if (batch == 0) return PJX_OK;
  if (kv_len == 0)
    return write_keyless(o, lse, (size_t)(batch * q_len * heads * v_dim), false, (size_t)(batch * heads * q_len), s,
                         "pjx_mla_decode");
  a.f16 = dtype == PJX_DTYPE_F16;
  // the latent is K and V at once: capacity B * S * R 16-bit values
  const bool streamed = decode_streams_kv(batch * kv_len * rank * 2, kStreamBytesLatent);
  return a.f16 ? run_mla_h16<F16Fmt>(a, rank, v_dim, streamed, workspace, workspace_bytes, s)
               : run_mla_h16<Bf16Fmt>(a, rank, v_dim, streamed, workspace, workspace_bytes, s);
}
