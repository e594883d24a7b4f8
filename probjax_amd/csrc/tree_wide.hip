// Tree attention for drafts of many rows (tree_decode.hip takes few): 16 bits,
// head dims 64 and 128.  With R = (Hq/Hkv)*T rows a key costs 4 D R operations
// and 4 D bytes, so from some 64 rows on the key loop is a flash forward's: one
// workgroup owns 32 RW rows and a chunk of keys, whose K and V tiles all of its
// RW KG waves share in LDS.  Each wave owns 32 rows (KG waves the same ones: they
// take different 32-key blocks of a tile and are joined at the end); the scores of
// the next tile are formed beside this one's exponentials.  The narrow kernel gives
// each wave keys of its own and all rows, 16 at a time: it reads K and V without
// LDS, but its accumulators of 64 rows leave one wave per SIMD, and every further
// 64 rows read the cache again (1 / 16 / 8 sequences of the table at the launch:
// 55 / 128 / 296 us for 18 / 68 / 50).
//
// Row groups of one work item are placed 8 workgroups apart, on one XCD, whose
// L2 gives all but the first their K and V (HBM traffic of 244 rows, two groups:
// that of one).  Bound by latency on one sequence (launch, lengths, first tile and
// four tiles in turn, 1 us each: 15 us), by HBM on 16 (285 MB in 70 us, 4.1 TB/s), on
// the widest by a tile's work on each SIMD and in LDS, about 1000 cycles each of
// matrix instructions, exponentials and reads for the 2500 that a tile takes.
// The weights p enter their product with V rounded to the 16-bit type, as the flash
// forward's do; scores, sums and outputs are float32 until the last store.
#include "decode_common.h"
#include "flash_common.h"

namespace pjx {

constexpr int kWideKeys = 64;  // keys of a tile

// The 32 keys from slot j behind the prefix's end on that token t sees, as bits.
__device__ __forceinline__ uint32_t tree_bits(const TreeTable& tt, int t, int j) {
  auto word = [&](int i) { return (unsigned)i < (unsigned)kTreeWords ? tt.bits[t][i] : 0u; };
  if (j <= -32) return 0xffffffffu;
  if (j < 0) return word(0) << -j | ((1u << -j) - 1u);
  const int s = j & 31;
  return s ? word(j >> 5) >> s | word((j >> 5) + 1) << (32 - s) : word(j >> 5);
}

template <typename E, int D, int RW, int KG>
__global__ __launch_bounds__(64 * RW * KG, 2) void tree_wide_kernel(DecodeArgs a, int groups) {
  using T = Bf16Tile<D>;
  constexpr int BK = T::BK, ROWB = T::ROWB, TILE_B = T::TILE_B;
  constexpr int NB = BK / 32 / KG;        // 32-key blocks of a wave's tile
  constexpr int NW = RW * KG, RPW = BK / NW;  // waves, rows of a tile that each loads
  constexpr int NLD = RPW / T::RPI;
  static_assert(BK == kWideKeys && NB >= 1 && NLD * T::RPI == RPW, "tile");
  // (objects of their own: the compiler waits for every load in flight before it
  // reads an object that one of them writes)
  __shared__ __attribute__((aligned(1024))) unsigned char k_lds0[TILE_B], k_lds1[TILE_B], v_lds0[TILE_B], v_lds1[TILE_B];
  __shared__ TreeTable tree;
  __shared__ int sched[4 + 2 * kSchedMaxBatch];

  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rw = w % RW, kg = w / RW;
  const int col = lane & 31, half = lane >> 5;
  const int rg = blockIdx.x / 8 % groups, item = blockIdx.x / (8 * groups) * 8 + blockIdx.x % 8;
  int b, g, chunk_id, L;
  if (!decode_item(a, sched, b, g, chunk_id, L, item)) return;
  const int c0 = chunk_id * a.chunk, c1 = min(c0 + a.chunk, L);
  const int P = prefix_len(a, b);
  const int rdim = a.orow;
  // Loads: the tile's first token is the buffer's base, so offsets within a tile
  // stay below 64 token strides (the launcher checks 32 bits).
  const uint32_t krow = (uint32_t)a.k_t * 2, vrow = (uint32_t)a.v_t * 2;
  const unsigned char* Kb = (const unsigned char*)(a.k + b * a.k_b + g * a.k_h);
  const unsigned char* Vb = (const unsigned char*)(a.v + b * a.v_b + g * a.v_h);
  uint32_t voffK[NLD], voffV[NLD];
#pragma unroll
  for (int j = 0; j < NLD; ++j) {
    const int r = RPW * w + T::RPI * j + lane / T::NC, slot = lane % T::NC;
    voffK[j] = row_chunk(r, krow, slot ^ T::swz_k(r), rdim);
    voffV[j] = row_chunk(r, vrow, slot ^ T::swz_v(r), rdim);
  }
  f32x16 acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = f32x16{};
  float m_run = kMaxInit, l_run = 0.f;

  const int n_tiles = (c1 - c0 + BK - 1) / BK;
  auto issue = [&](const unsigned char* base, int64_t stride, uint32_t row_b, const uint32_t* voff, int t,
                   unsigned char* dst) {
    if (t >= n_tiles) return;
    const int k0 = c0 + t * BK, nvalid = min(BK, c1 - k0);
    const rsrc_t rs = make_rsrc(base + (size_t)k0 * stride * 2, (uint32_t)(nvalid - 1) * row_b + rdim * 2);
#pragma unroll
    for (int j = 0; j < NLD; ++j) buffer_load_lds16(rs, dst + (RPW * w + T::RPI * j) * ROWB, voff[j]);
  };
  auto issue_k = [&](int t, unsigned char* dst) { issue(Kb, a.k_t, krow, voffK, t, dst); };
  auto issue_v = [&](int t, unsigned char* dst) { issue(Vb, a.v_t, vrow, voffV, t, dst); };

  // Tile t lives in stage t % 2; K is loaded one tile ahead of V.  The first tile
  // comes while the queries do and the table is built.
  issue_k(0, k_lds0);
  issue_v(0, v_lds0);
  issue_k(1, k_lds1);
  const int row = rg * 32 * RW + 32 * rw + col;
  const bool row_in = row < a.rows;
  int tok = 0, h = 0;
  if (row_in) row_to_head(a, g, row, tok, h);
  typename E::v8 qf[D / 16];
  {
    const uint16_t* qrow = a.q + ((size_t)(b * a.Lq + tok) * a.Hq + h) * rdim;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      u32x4 raw = {0u, 0u, 0u, 0u};
      if (row_in && 16 * s + 8 * half < rdim) raw = *(const u32x4*)(qrow + 16 * s + 8 * half);
      qf[s] = E::as8(raw);
    }
  }

  if (c1 > P) build_tree<NW>(a, b, tree);

  uint32_t offK[D / 16];
#pragma unroll
  for (int st = 0; st < D / 16; ++st) offK[st] = col * ROWB + 16 * ((2 * st + half) ^ T::swz_k(col));
  uint32_t offV[D / 32];
  {
    const int s16 = lane & 15, grp = lane >> 4;
    const int r = 4 * half + s16 / 4;
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      const int chunk = 4 * db + 2 * (grp & 1) + ((s16 & 3) >> 1);
      offV[db] = r * ROWB + 16 * (chunk ^ T::swz_v(r)) + 8 * (s16 & 1);
    }
  }

  auto scores = [&](const unsigned char* ks, f32x16* s) {
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
      s[kb] = f32x16{};
#pragma unroll
      for (int st = 0; st < D / 16; ++st) {
        const typename E::v8 kf = E::as8(*(const u32x4*)(ks + (kg * NB + kb) * 32 * ROWB + offK[st]));
        s[kb] = E::mma32(kf, qf[st], s[kb]);
      }
    }
  };
  // Tile t's softmax and products with V, and beside them the scores of tile t + 1
  // (of whatever its slot holds past the last tile).
  auto compute = [&](int t, f32x16* s, unsigned char* vs, const unsigned char* next, f32x16* sn) {
    const int k0 = c0 + t * BK;
    const bool tail = k0 + BK > P;
    bool unbounded = false;  // as in gqa_decode
    if (tail) {
      bool any = false;
#pragma unroll
      for (int i = 0; i < TILE_B / (16 * 64 * NW); ++i) {
        u32x4* p = (u32x4*)(vs + 16 * (tid + 64 * NW * i));
        u32x4 x = *p;
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t y = finite_halves<E>(x[e]);
          odd |= y != x[e];
          x[e] = y;
        }
        if (odd) *p = x;
        any |= odd;
      }
      unbounded = __syncthreads_or(any);
    }
    // Register r of block kb holds key k0 + 32 (kg NB + kb) + 8 (r / 4) + 4 half + r % 4.
    if (tail || k0 + BK > c1) {
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        const int kk = k0 + 32 * (kg * NB + kb), left = c1 - kk;
        uint32_t sees = tree_bits(tree, tok, kk - P);
        if (left < 32) sees &= left <= 0 ? 0u : (1u << left) - 1u;
        sees >>= 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!(sees >> (8 * (r >> 2) + (r & 3)) & 1u)) s[kb][r] = -INFINITY;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; r += 2) mx = fmaxf(mx, fmaxf(s[kb][r], s[kb][r + 1]));
    const float mc = xor32_max(mx) * a.cx;
    if (wave_any(mc > m_run + kRescaleLog2)) {
      const float m_new = fmaxf(m_run, mc);
      const float corr = fast_exp2(m_run - m_new);
      m_run = m_new;
      l_run *= corr;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= corr;
    }
    scores(next, sn);
    float rs0 = 0.f, rs1 = 0.f;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = fast_exp2(fmaf(s[kb][r], a.cx, -m_run));
        const float p1 = fast_exp2(fmaf(s[kb][r + 1], a.cx, -m_run));
        rs0 += p0;
        rs1 += p1;
        s[kb][r] = p0;
        s[kb][r + 1] = p1;
      }
    l_run += rs0 + rs1;
    typename E::v8 pf[2 * NB];
#pragma unroll
    for (int c = 0; c < 2 * NB; ++c) {
      u32x4 pk;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        pk[j] = E::pack2(s[c >> 1][8 * (c & 1) + 2 * j], s[c >> 1][8 * (c & 1) + 2 * j + 1]);
      pf[c] = E::as8(pk);
    }
    const unsigned char* vw = vs + kg * NB * 32 * ROWB;
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
#pragma unroll
      for (int c = 0; c < 2 * NB; ++c) {
        const u32x2 lo = lds_read_tr16(vw + 16 * c * ROWB + offV[db]);
        const u32x2 hi = lds_read_tr16(vw + (16 * c + 8) * ROWB + offV[db]);
        const u32x4 av = {lo[0], lo[1], hi[0], hi[1]};
        acc[db] = E::mma32(E::as8(av), pf[c], acc[db]);
      }
    }
    if (unbounded) {
      // p * v for the infinite and NaN elements, key by key, for the rows that see it
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        const int kk = k0 + 32 * (kg * NB + kb);
        const uint32_t sees = tree_bits(tree, tok, kk - P);
#pragma unroll 1
        for (int i = 0; i < min(32, c1 - kk); ++i) {
          float p = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) p = r == (i & 3) + 4 * (i >> 3) ? s[kb][r] : p;
          p = __shfl(p, col + 32 * (i >> 2 & 1));
          const uint16_t* vr = (const uint16_t*)Vb + (int64_t)(kk + i) * a.v_t + 4 * half;
#pragma unroll
          for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if (32 * db + 8 * q >= rdim) continue;
              const u32x2 u = *(const u32x2*)(vr + 32 * db + 8 * q);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t diff = u[e] ^ finite_halves<E>(u[e]);
                if ((sees >> i & 1u) && (diff & 0xffffu)) acc[db][4 * q + 2 * e] = fmaf(p, E::lo(u[e]), acc[db][4 * q + 2 * e]);
                if ((sees >> i & 1u) && (diff >> 16)) acc[db][4 * q + 2 * e + 1] = fmaf(p, E::hi(u[e]), acc[db][4 * q + 2 * e + 1]);
              }
            }
        }
      }
    }
  };

  f32x16 sa[NB], sb[NB];
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  scores(k_lds0, sa);
  // Iteration t: K of tile t + 1 and V of tile t have landed; K of tile t + 2 takes
  // the place of tile t's, V of tile t + 1 that of tile t - 1's.
  for (int t = 0; t < n_tiles; t += 2) {
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    issue_k(t + 2, k_lds0);
    issue_v(t + 1, v_lds1);
    compute(t, sa, v_lds0, k_lds1, sb);
    if (t + 1 >= n_tiles) break;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    issue_k(t + 3, k_lds1);
    issue_v(t + 2, v_lds0);
    compute(t + 1, sb, v_lds1, k_lds0, sa);
  }

  if constexpr (KG > 1) {
    // Waves of the same rows: the second hands (max, sum, O) to the first
    // through LDS, in the same register layout.
    static_assert(KG == 2 && RW <= 4 && (D / 32) * 4 * 64 * 16 == TILE_B && RW * 64 * 8 <= sizeof(TreeTable),
                  "hand-over");
    __syncthreads();
    // (each wave's O in a tile's place of its own, (max, sum) in the table's)
    unsigned char* own = rw == 0 ? v_lds0 : rw == 1 ? v_lds1 : rw == 2 ? k_lds0 : k_lds1;
    f32x4* xo = (f32x4*)own + lane;
    float* xml = (float*)&tree + 2 * (rw * 64 + lane);
    if (kg == 1) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
          xo[(4 * i + r / 4) * 64] = f32x4{acc[i][r], acc[i][r + 1], acc[i][r + 2], acc[i][r + 3]};
      xml[0] = m_run;
      xml[1] = l_run;
    }
    __syncthreads();
    if (kg == 1) return;
    const float m1 = xml[0], l1 = xml[1], M = fmaxf(m_run, m1);
    const float f0 = fast_exp2(m_run - M), f1 = fast_exp2(m1 - M);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const f32x4 o1 = xo[(4 * i + r / 4) * 64];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][r + j] = fmaf(acc[i][r + j], f0, o1[j] * f1);
      }
    l_run = fmaf(l_run, f0, l1 * f1);
    m_run = M;
  }
  if (!row_in) return;
  float l_tot = xor32_sum(l_run);
  if (!tree_token(a, b, tok)) {  // a row without a valid key
    m_run = kMaxInit;
    l_tot = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = f32x16{};
  }
  if (c0 == 0 && L <= a.chunk) {
    const bool some = some_key(l_tot);
    const float inv = some ? 1.f / l_tot : 0.f;
    uint16_t* orow = a.o + ((size_t)(b * a.Lq + tok) * a.Hq + h) * rdim;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (db * 32 + 8 * q >= rdim) continue;
        const u32x2 pk = {E::pack2(acc[db][4 * q] * inv, acc[db][4 * q + 1] * inv),
                          E::pack2(acc[db][4 * q + 2] * inv, acc[db][4 * q + 3] * inv)};
        *(u32x2*)(orow + db * 32 + 8 * q + 4 * half) = pk;
      }
    if (a.lse && half == 0)
      a.lse[((size_t)b * a.Hq + h) * a.Lq + tok] = some ? (m_run + __log2f(l_tot)) * kLn2 : INFINITY;
  } else {
    const size_t at = ((size_t)(b * a.G + g) * a.nch + chunk_id) * a.rows + row;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(f32x4*)(a.ws_o + at * a.dv + db * 32 + 8 * q + 4 * half) =
            f32x4{acc[db][4 * q], acc[db][4 * q + 1], acc[db][4 * q + 2], acc[db][4 * q + 3]};
    if (half == 0) {
      a.ws_ml[2 * at] = m_run;
      a.ws_ml[2 * at + 1] = l_tot;
    }
  }
}

// (one item per sequence and head: the chunk kernel wrote every row)
template <typename E, int D, int RW, int KG>
static int launch_wide(DecodeArgs& a, void* ws, size_t ws_bytes, hipStream_t s, const char* who) {
  if (!ws || ws_bytes < ws_size(a.B, a.G, a.rows, a.Lk, a.dv, a.chunk))
    return fail(PJX_ERR_WORKSPACE, "tree decode: workspace missing or too small");
  a.ws_o = (float*)ws;
  a.ws_ml = a.ws_o + (size_t)a.B * a.G * a.nch * a.rows * a.dv;
  const int64_t items = (int64_t)a.B * a.G * a.nch, groups = (a.rows + 32 * RW - 1) / (32 * RW);
  const int64_t blocks = (items + 7) / 8 * 8 * groups;
  if (blocks > 0xffffffffLL / (64 * RW * KG) || (int64_t)a.B * a.G * a.rows > 0x7fffffffLL)
    return fail(PJX_ERR_INVALID, "tree decode: grid too large");
  launch_kernel<tree_wide_kernel<E, D, RW, KG>>(dim3((unsigned)blocks), dim3(64 * RW * KG), 0, s, a, (int)groups);
  const int rc = check_launch(who);
  if (rc || a.nch == 1) return rc;
  return a.nch <= kFewChunks ? launch_merge_few(a, s, who) : launch_decode_merge(a, s, who);
}

template <typename E>
static int run_wide(DecodeArgs& a, int d, int rw, void* ws, size_t n, hipStream_t s, const char* who) {
  if (d == 64)
    return rw == 2 ? launch_wide<E, 64, 2, 2>(a, ws, n, s, who) : launch_wide<E, 64, 4, 2>(a, ws, n, s, who);
  return rw == 2 ? launch_wide<E, 128, 2, 2>(a, ws, n, s, who) : launch_wide<E, 128, 4, 2>(a, ws, n, s, who);
}

bool tree_wide_takes(const DecodeArgs& a, int head_dim, bool f32) {
  return !f32 && head_dim <= 128 && a.rows > 32 && std::max(a.k_t, a.v_t) <= (int64_t)1 << 24;
}

int run_tree_wide(DecodeArgs& a, int head_dim, bool auto_chunk_size, void* ws, size_t ws_bytes, hipStream_t s,
                  const char* who) {
  // 128 rows a workgroup (of eight waves), unless they are fewer or would leave the
  // device idle; else 64 (of four).  Chunks from 256 keys on, doubled while some
  // workgroups per CU remain, one of eight waves or two of four: every chunk's
  // partial results cost as much traffic as a key a row, written and read again.
  // MI355X, us, chunk 256 / 512 / 1024 / 2048 / 4096, 8 KV heads of 128:
  //   1 x 4096, 104 rows               64 rows 18 / 20 / 26 / 39 / 65   128 rows 20 / 22 / 28 / 44 / 73
  //   16 x 512 .. 8192 keys, 64 rows   64 rows 103 / 88 / 75 / 68 / 90
  //   8 x 1500 .. 4096 keys, 244 rows  64 rows 92 / 70 / 58 / 50 / 67   128 rows 105 / 74 / 63 / 50 / 75
  //   8 x 4096, 244 rows, the chunk as chosen: 64 rows 56, 128 rows 52; 8 x 2048, 1024 rows: 119, 105
  const int64_t pairs = (int64_t)a.B * a.G;
  const int rw = a.rows <= 64 || pairs * ((a.Lk + 511) / 512) * ((a.rows + 127) / 128) < 512 ? 2 : 4;
  if (auto_chunk_size) {
    const int64_t work = pairs * a.Lk * ((a.rows + 32 * rw - 1) / (32 * rw)), most = rw == 2 ? 640 : 320;
    int64_t c = std::max(a.chunk, 256);
    while (c < 2048 && work / c > most) c *= 2;
    a.chunk = (int)c;
    a.nch = (int)std::max<int64_t>((a.Lk + c - 1) / c, 1);
  }
  return a.f16 ? run_wide<F16Fmt>(a, head_dim, rw, ws, ws_bytes, s, who)
               : run_wide<Bf16Fmt>(a, head_dim, rw, ws, ws_bytes, s, who);
}

}  // namespace pjx
