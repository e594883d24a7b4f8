// Attention of each sequence's newest tokens over a paged KV cache for gfx950, in the
// cache's own type or over 8 bits:
//   o_t = sum_j softmax_j(scale q_t.k_j) v_j,  j < L - (T-1-t),
// L keys of the sequence, T new tokens (one as a rule).
//
// A wave takes a share of the keys of all sequences, laid end to end in steps of 32, for
// one KV head, with its (Hq/Hkv)*T packed query rows as the columns of the matrix
// instructions (NRB blocks of 16).  Shares are equal whatever the lengths, and as many as
// the device holds waves: each compute unit streams the same bytes at the same time (parts
// of whole sequences left the last units 82 us for a share that the first had in 58).  A
// share that runs into the next sequence leaves a partial result and goes on; a second
// kernel joins the parts of a sequence.  What a share is follows from the lengths, which
// only the device knows: every wave works it out from all of them, so a grid made for the
// capacity, or captured once, is shared by whatever keys there are.  A workgroup's
// waves are neighbouring heads on the same keys, so rows that lie side by side are read
// side by side (8-bit rows of 64 features, [page, H, D]: 43 us against 58 as workgroups of
// their own).
//
// A wave's K and V rows go from memory to LDS by loads of 16 bytes a lane that no
// register waits for, whole rows each, one step ahead.  The lanes look up a page each,
// once per key, and hand the rows' addresses around in LDS, so pages of any size and order
// cost the same.  K rows are read back as the matrix operand; V is transposed by the LDS
// reads (ds_read_b64_tr).
// 8-bit rows stay codes until they are operands, exact in bf16 and fp16; their powers of
// two go to the scores (K) and to the softmax weights (V), after and before the products.
//
// Bound by HBM where there is much to read, 32 query on 8 KV heads of 128: 32 x 512-8192
// keys in bf16 571 MB in 92 us (87 of them the first kernel, 6.5 TB/s), in 8 bits 288 MB in
// 51; 131072 keys of one sequence 271 MB in 49.  By its chain of loads (lengths, pages,
// rows), ~5 us, and the second kernel's, ~4, where there is little: 4096 keys in 11.
// The hint on the loads that rows are not read again (nt) matters most: 98 us against 165
// without it behind other work that filled the caches (8 bits 63 against 106), though a
// cache of 67-84 MB read over and over by itself would take 24-31 us for 30-33 without.
// With several groups of rows, each of which reads all keys, it is mixed: 128 rows (four
// groups of 32) of 4 KV heads of 128, 32 x 512-8192 bf16 keys, 124 us with it and 132
// without, 128 rows of 256 features (eight groups of 16, 587 MB) 438 and 309.
#include <stdio.h>

#include "pages.h"

namespace pjx {

// Keys of a share at least: 64, but of float32 tokens 32 (a step; of a float32 cache's rows
// of 256 features two), since their products take as long as the loads.  It counts where
// there are few keys.  512 keys, 16 query on 4 KV heads of 64 / 128 / 256, us in a captured
// graph with 32 and with 64: float32 8.6, 10.0 / 11.0, 13.5 / 14.7, 20.1; float32 over 8
// bits 10.1, 12.7 / 10.5, 13.2 / 14.5, 19.7; bf16 7.5, 8.2 / 8.3, 9.4 / 10.2, 11.5; bf16
// over 8 bits 8.0, 9.0 / 8.2, 9.1 / 9.5, 10.7.  So one step would be faster in 16 bits too,
// by 1 us of a call that the host takes 11 for.
template <typename E>
constexpr int least_share() {
  return std::is_same<E, F32Fmt>::value ? 32 : 64;
}

struct PagedArgs {
  PageArgs p;
  const char* q;
  char* o;
  float* lse;
  const int32_t* lengths;
  float* ws_o;   // [shares + B][H][rows][W] unnormalised outputs of the parts
  float* ws_ml;  // [shares + B][H][rows][2] running max (log2 units), sum
  int B, T, Hq, D, rows;
  int shares;    // of a KV head, at most
  int least;     // steps of a share at least
  int step_log;  // keys of a step, as a power of two
  int slices;    // paged_join_kernel
  FastDiv by_g, by_t, by_shares;
  float cx;      // sm_scale * log2(e)
};

__device__ __forceinline__ int paged_len(const PagedArgs& a, int b) {
  const int room = a.p.most * a.p.page;
  return a.lengths ? min(max(a.lengths[b], 0), room) : room;
}

// The steps of all sequences, end to end, and a share of them.  Lane l knows sequence l's
// length (0 behind the last) and the steps up to its end.
__device__ __forceinline__ int steps_of(const PagedArgs& a, int L) { return (L + (1 << a.step_log) - 1) >> a.step_log; }
struct Lane {
  int len, upto;
};
__device__ __forceinline__ Lane lane_steps(const PagedArgs& a) {
  const int lane = threadIdx.x & 63, L = lane < a.B ? paged_len(a, lane) : 0;
  return {L, wave_scan(steps_of(a, L))};
}
// The sum over the lanes' sequences behind the first 64 and before `end`, in all lanes.
__device__ __forceinline__ int later_steps(const PagedArgs& a, int end) {
  int n = 0;
#pragma unroll 8
  for (int b0 = 64; b0 < end; b0 += 64) {
    const int b = b0 + (threadIdx.x & 63), L = paged_len(a, min(b, a.B - 1));
    n += b < end ? steps_of(a, L) : 0;
  }
  return __builtin_amdgcn_readlane(wave_scan(n), 63);
}
__device__ __forceinline__ int all_steps(const PagedArgs& a, const Lane& s) {
  const int all = __builtin_amdgcn_readlane(s.upto, 63);
  return a.B <= 64 ? all : all + later_steps(a, a.B);
}
__device__ __forceinline__ int share_of(const PagedArgs& a, int all) { return max(a.by_shares(all + a.shares - 1), a.least); }

// A step of a wave: keys k0 .. of sequence b, which has `len`; `left` steps of the share
// from this one on.
struct Cursor {
  int b, k0, len, left;
};
// Step `at` of all steps.
__device__ __forceinline__ Cursor find_step(const PagedArgs& a, const Lane& s, int at) {
  const int lane = threadIdx.x & 63;
  int L = s.len, upto = s.upto;
  for (int b0 = 0;;) {
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > at);
    if (past) {
      const int src = __builtin_ctzll(past), len = __builtin_amdgcn_readlane(L, src);
      const int before = __builtin_amdgcn_readlane(upto, src) - steps_of(a, len);
      return {b0 + src, (at - before) << a.step_log, len, 0};
    }
    const int run = __builtin_amdgcn_readlane(upto, 63);
    b0 += 64;
    if (b0 >= a.B) return {0, 0, 0, 0};
    L = b0 + lane < a.B ? paged_len(a, b0 + lane) : 0;
    upto = run + wave_scan(steps_of(a, L));
  }
}
// The next step of the share; its last one stays (with left = 0).  lens: lane l's length.
__device__ __forceinline__ Cursor next_step(const PagedArgs& a, int lens, Cursor c) {
  if (c.left <= 1) return {c.b, c.k0, c.len, 0};
  c.left -= 1;
  c.k0 += 1 << a.step_log;
  if (c.k0 >= c.len) {
    c.k0 = 0;
    do {  // (a step is left, so a sequence follows that has keys)
      c.b += 1;
      c.len = c.b < 64 ? __builtin_amdgcn_readlane(lens, c.b) : __builtin_amdgcn_readfirstlane(paged_len(a, c.b));
    } while (c.len == 0);
  }
  return c;
}
// Steps before those of sequence b, and b's.
__device__ __forceinline__ int steps_before(const PagedArgs& a, const Lane& s, int b, int& n_b) {
  if (b < 64) {
    n_b = steps_of(a, __builtin_amdgcn_readlane(s.len, b));
    return __builtin_amdgcn_readlane(s.upto, b) - n_b;
  }
  n_b = steps_of(a, __builtin_amdgcn_readfirstlane(paged_len(a, b)));
  return __builtin_amdgcn_readlane(s.upto, 63) + later_steps(a, b);
}

// A step's K or V rows in LDS: rows of W elements of C, their 16-byte chunks at chunk ^
// swz(row).  So that no read meets in a bank: a matrix operand of K (16 rows at one chunk
// for 16 lanes, the next for the following 16), and the transposing reads of V (8 rows at
// two chunks, 16 rows of codes at one).
template <typename C, int W>
struct PageTile {
  static constexpr int CS = fmt_size<C>(), ROWB = W * CS, NC = ROWB / 16;
  static constexpr int KS = ROWB > 512 ? 16 : 32;  // keys of a step
  static constexpr int BYTES = KS * ROWB;
  static constexpr int NL = BYTES / 1024;          // loads of a wave
  static constexpr int RPI = 64 / NC;              // rows of a load
  __device__ __forceinline__ static constexpr int swz(int r) {
    return NC == 4 ? ((r >> 2) ^ ((r >> 4) << 1)) & 3 : NC == 8 ? (r & 6) | ((r >> 4) & 1) : ((r & 7) << 1) | ((r >> 4) & 1);
  }
  __device__ __forceinline__ static int at(int r, int chunk) { return r * ROWB + 16 * (chunk ^ swz(r)); }
};

// Loads from an address of each lane's own into LDS: lane l's 16 bytes land at lds + 16 * l
// (dword or byte: at lds + 4 * l).  Written in assembly (they have no result a register
// waits for): the compiler makes every transposing read of LDS wait for all loads it knows
// of.  So it knows of none in the key loop, where arrived() counts them.  (M0 is not
// in the clobbers, which may not name it; nothing else here uses it.)
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p);
}
__device__ __forceinline__ void load_lds16(uint64_t from, uint32_t lds) {
  lds = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(from), "s"(lds) : "memory");
}
__device__ __forceinline__ void load_lds4(uint64_t from, uint32_t lds) {
  lds = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(lds) : "memory");
}
__device__ __forceinline__ void load_lds1(uint64_t from, uint32_t lds) {
  lds = __builtin_amdgcn_readfirstlane(lds);
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_ubyte %0, off" ::"v"(from), "s"(lds) : "memory");
}

// This wave's LDS accesses so far are done, and stay before this point.
__device__ __forceinline__ void lds_done() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(15 | (7 << 4) | (0 << 8) | (3 << 14));  // lgkmcnt(0)
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// All of this wave's loads but the last N have arrived.
template <int N>
__device__ __forceinline__ void arrived() {
  __builtin_amdgcn_sched_barrier(0);
  wait_vmcnt<N>();
  __builtin_amdgcn_sched_barrier(0);
}

// x, as the compiler cannot know it: what is made of it is made where it is used, and not
// kept in registers through a loop that seldom comes there.
__device__ __forceinline__ int once(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

__device__ __forceinline__ uint32_t bits_of(float x) {
  uint32_t u = __float_as_uint(x);
  asm volatile("" : "+v"(u));  // (the sources are compiled without NaN in mind)
  return u;
}

// Whether any element of N x 4 dwords of floats C is infinite or NaN.
template <typename C, int N>
__device__ __forceinline__ bool any_odd(const u32x4 (&x)[N]) {
  if constexpr (std::is_same<C, F32Fmt>::value) {
    bool odd = false;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) odd |= (x[i][e] & 0x7f800000u) == 0x7f800000u;
    return odd;
  } else {  // by the largest magnitude, two elements at a time
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[i][e] & 0x7fff7fffu));
    return max((uint32_t)m[0], (uint32_t)m[1]) >= (C::kF16 ? 0x7c00u : 0x7f80u);
  }
}
// Whether any of a dword's 4 codes is NaN.
__device__ __forceinline__ bool odd_codes(uint32_t x) {
  const uint32_t y = ~x & 0x7f7f7f7fu;  // a byte is 0 where the code is NaN
  return ((y - 0x01010101u) & ~y & 0x80808080u) != 0u;
}

// 8 codes as an operand of E (bf16 or fp16).
template <typename E>
__device__ __forceinline__ typename E::v8 codes8(uint32_t lo, uint32_t hi) {
  u32x4 r;
  if constexpr (E::kF16) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true));
  }
  return E::as8(r);
}
__device__ __forceinline__ f32x4 codes4(uint32_t w) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return f32x4{lo[0], lo[1], hi[0], hi[1]};
}

// Waves of a compute unit at a time: four, one to a SIMD and with 64 rows each on their
// way, keep the memory busy from rows of 128 bytes on (32 x 512-8192 keys of 8 heads of 128
// in 8 bits: 51 us with four, 53 with eight, 57 and more where units hold different numbers
// of them); eight on shorter ones (the same of 64 features: 34 us against 51, head-major
// pages 31 against 49).
template <typename C, int W>
constexpr int paged_waves() {
  return W * fmt_size<C>() >= 128 ? 4 : 8;
}
constexpr int kPagedWaves = 8;  // of a compute unit at most
// Waves of a workgroup: those of rows that together make up 512 bytes and more of a token,
// if its heads lie side by side (64 features in 8 bits, 32 x 512-8192 keys: 36 us with
// eight, 38 with four, 45 with two).
template <typename C, int W>
constexpr int paged_group() {
  return W * fmt_size<C>() >= 128 ? 4 : 8;
}
// Waves of a SIMD that the registers are to leave room for (256 features, and float32 sums
// of more than 64, need more than half of them).
template <typename C, typename E, int W>
constexpr int paged_occupancy() {
  return W == 256 || (std::is_same<E, F32Fmt>::value && W > 64) ? 1 : 2;
}

// Waves of a workgroup that has a whole sequence (WHOLE): as many as its LDS and registers
// allow.
template <typename C, typename E, int W, int NRB>
constexpr int paged_whole_waves() {
  return W * fmt_size<C>() > 256 || W == 256 || (W > 64 && (std::is_same<E, F32Fmt>::value || NRB > 1)) ? 4 : 8;
}

// What the chunks behind a row's end are loaded from.
__device__ const __attribute__((aligned(16))) uint32_t kZeros[4] = {};

// C: format of the cache, E: of q and o; W: features of a row in LDS (64, 128, 256), ROWS:
// a row has fewer, and zeros behind them; NRB: blocks of 16 query rows.  WHOLE: a workgroup
// takes one sequence's keys for a KV head, an equal number of steps to each of its waves,
// and joins them itself.
template <typename C, typename E, int W, int NRB, bool ROWS, bool WHOLE>
__global__ __launch_bounds__(64 * (WHOLE ? paged_whole_waves<C, E, W, NRB>() : paged_group<C, W>()), (paged_occupancy<C, E, W>())) void paged_decode_kernel(PagedArgs a) {
  using T = PageTile<C, W>;
  constexpr bool F32 = std::is_same<E, F32Fmt>::value, QUANT = std::is_same<C, E4m3Fmt>::value;
  // The weights enter their product with V in 16 bits, in two parts: rounded to the type,
  // and the rounding's rest.  That leaves the output's own rounding (without the second
  // part errors are 1.3 times it) and costs nothing where the memory is waited for.  Codes
  // take them as bf16 whatever E is: their rows' powers of two have its range, not fp16's.
  typedef typename std::conditional<QUANT && !F32, Bf16Fmt, E>::type EV;
  // fp16 ends at 2^-24: behind a key that has nearly all of the weight (and, as a rule, a
  // value near 0) the others' would be lost.  So its weights are taken relative to the
  // largest of their own step (per row), the first part times 2^15, the rest times 2^27 (it
  // is at most 2^-12 of that largest), and what the step adds is scaled to the running
  // maximum in float32.  A weight is then off by at most 2^-22 of itself, or 2^-52 of its
  // step's largest: over all steps that is less than 32 * 2^-52 * 65504 < 2^-31 of an
  // output, whose own steps are 2^-24 and more.  (32 x 512-8192 keys of 8 heads of 128, one
  // token: 90.5 us with and without; 64 tokens of 8 x 512-4096, bound by the products: 79
  // for 71.)
  constexpr bool STEP_MAX = std::is_same<EV, F16Fmt>::value;
  constexpr float kUp = 32768.f, kRestUp = 4096.f;
  constexpr int KS = T::KS, KB = KS / 16, NL = T::NL, CS = T::CS, ES = fmt_size<E>();
  constexpr int NDB = W / 16;
  constexpr int NW = WHOLE ? paged_whole_waves<C, E, W, NRB>() : paged_group<C, W>();
  __shared__ __attribute__((aligned(1024))) unsigned char k_lds[NW * T::BYTES];
  __shared__ __attribute__((aligned(1024))) unsigned char v_lds[NW * T::BYTES];
  __shared__ __attribute__((aligned(16))) uint64_t rows_lds[NW * 64];  // addresses of a step's K, V rows
  __shared__ __attribute__((aligned(16))) uint32_t exp_lds[QUANT ? NW * 64 : 4];
  __shared__ __attribute__((aligned(16))) uint32_t page_lds[NW * 64];  // pages of the next step's keys
  __shared__ float2 ml_lds[WHOLE ? NW * 16 : 1];
  const PageArgs& p = a.p;
  const int lane = threadIdx.x & 63, c16 = lane & 15, q4 = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int share = 0, g, lens = 0;
  Cursor cur;
  if constexpr (WHOLE) {
    cur.b = a.by_g(blockIdx.x);
    g = blockIdx.x - cur.b * p.H;
    cur.len = __builtin_amdgcn_readfirstlane(paged_len(a, cur.b));
    const int steps = steps_of(a, cur.len), per = (steps + NW - 1) / NW;
    cur.k0 = (w * per) * KS;
    cur.left = min(per, steps - w * per);
  } else {
    const int item = blockIdx.x * NW + w;
    share = a.by_g(item);
    g = item - share * p.H;
    const Lane steps = lane_steps(a);
    lens = steps.len;
    const int all = all_steps(a, steps), size = share_of(a, all);
    if ((int64_t)share * size >= all) return;
    cur = find_step(a, steps, share * size);
    cur.left = min(size, all - share * size);
  }
  Cursor nxt = next_step(a, lens, cur), then = next_step(a, lens, nxt);
  const int row0 = blockIdx.y * 16 * NRB;

  unsigned char *kl = k_lds + w * T::BYTES, *vl = v_lds + w * T::BYTES;
  uint64_t* rl = rows_lds + w * 64;
  uint32_t *el = exp_lds + (QUANT ? w * 64 : 0), *pl = page_lds + w * 64;
  const uint32_t kl_at = lds_offset(kl), vl_at = lds_offset(vl), el_at = lds_offset(el), pl_at = lds_offset(pl);

  // ---- the rows of a step, one lane per key and tensor (K: lanes 0..31, V: 32..63) ----
  const int half = lane >> 5, lk = lane & 31;
  const uint64_t pool = (uint64_t)(half ? p.v : p.k) + (uint64_t)g * (uint64_t)(half ? p.vh : p.kh);
  const int64_t page_step = half ? p.vp : p.kp, token_step = half ? p.vt : p.kt;
  const uint64_t exps = (uint64_t)(half ? p.ve : p.ke);
  auto look_up = [&](const Cursor& c) {  // the pages of a step's keys (without a table something else, unused)
    const uint64_t entry = p.table ? (uint64_t)(p.table + c.b * p.table_step) : (uint64_t)a.q;
    load_lds4(entry + 4ull * (uint32_t)(p.table ? p.by_page(min(c.k0 + (lk & (KS - 1)), c.len - 1)) : 0), pl_at);
  };
  uint64_t exp_at = 0;
  auto place = [&](const Cursor& c) -> uint32_t {  // their rows' addresses to LDS; which keys are there
    const uint32_t page = p.table ? pl[lane] : (uint32_t)c.b;
    const int key = c.k0 + (lk & (KS - 1)), kc = min(key, c.len - 1);
    const bool some = page < p.pages;
    const uint32_t pg = some ? page : 0u;
    const int slot = kc - p.by_page(kc) * p.page;
    rl[lane] = pool + (uint64_t)(pg * page_step + slot * token_step);
    if constexpr (QUANT) exp_at = exps + (uint64_t)((int64_t)(pg * (uint64_t)p.H + g) * p.page + slot);
    return (uint32_t)__builtin_amdgcn_ballot_w64(some && key < c.len) & (uint32_t)((1ull << KS) - 1);
  };
  const int row_chunks = a.D * CS / 16;
  auto fetch = [&](uint32_t to, int first) {
    uint64_t at[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) at[i] = rl[first + i * T::RPI + lane / T::NC];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int c = (lane % T::NC) ^ T::swz(i * T::RPI + lane / T::NC);
      load_lds16(!ROWS || c < row_chunks ? at[i] + 16 * c : (uint64_t)kZeros, to + 1024 * i);
    }
  };
  auto fetch_exps = [&]() {
    if constexpr (QUANT) load_lds1(exp_at, el_at);
  };

  // ---- a sequence: q as the B operand, features in the order the cache's rows are read in ----
  int lim[NRB];  // keys that the lane's row sees
  typename std::conditional<F32, f32x4, u32x4>::type qf[NRB][F32 ? W / 16 : W / 32];
  f32x4 acc[NRB][NDB];
  float m_run[NRB], l_run[NRB];
  bool from_start = false;
  auto begin = [&](const Cursor& c) {
    from_start = c.k0 == 0;
    const int r16 = once(c16), d4 = once(q4);
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
      const int row = row0 + 16 * rb + r16;
      const bool in = row < a.rows;
      const int gi = a.by_t(in ? row : 0), t = (in ? row : 0) - gi * a.T;
      lim[rb] = c.len - (a.T - 1 - t);
      const char* x = a.q + (((int64_t)c.b * a.T + t) * a.Hq + g * (a.Hq / p.H) + gi) * a.D * ES;
      if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < W / 16; ++j) {
          const int d = QUANT ? 64 * (j / 4) + 16 * d4 + 4 * (j % 4) : 16 * j + 4 * d4;
          qf[rb][j] = in && (!ROWS || d < a.D) ? *(const f32x4*)(x + 4 * d) : f32x4{};
        }
      } else {
#pragma unroll
        for (int j = 0; j < W / 32; ++j) {
          const int d = QUANT ? 64 * (j / 2) + 16 * d4 + 8 * (j % 2) : 32 * j + 8 * d4;
          qf[rb][j] = in && (!ROWS || d < a.D) ? *(const u32x4*)(x + 2 * d) : u32x4{0u, 0u, 0u, 0u};
        }
      }
      m_run[rb] = kMaxInit;
      l_run[rb] = 0.f;
#pragma unroll
      for (int i = 0; i < NDB; ++i) acc[rb][i] = f32x4{};
    }
    arrived<0>();  // (here, or the compiler waits for all loads at q's first use in every step)
  };

  auto begin_empty = [&]() {
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
      m_run[rb] = kMaxInit;
      l_run[rb] = 0.f;
#pragma unroll
      for (int i = 0; i < NDB; ++i) acc[rb][i] = f32x4{};
    }
  };

  uint32_t there = 0;
  const bool any = !WHOLE || cur.left > 0;
  if (any) {
    look_up(cur);
    begin(cur);
    there = place(cur);
    lds_done();
    look_up(nxt);
    fetch_exps();
    fetch(kl_at, 0);
    fetch(vl_at, 32);
  } else {
    begin_empty();
  }
  while (any) {
    const int k0 = cur.k0;
    arrived<NL>();  // K's rows and the next step's pages; behind them V's rows
    u32x4 kf[KB][T::NC / 4];  // chunk 4j + q4 of key 16kb + c16
    f32x4 ks[KB], vs[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int j = 0; j < T::NC / 4; ++j) kf[kb][j] = *(const u32x4*)(kl + T::at(16 * kb + c16, 4 * j + q4));
      if constexpr (QUANT) {
        const u32x4 ke = *(const u32x4*)(el + 16 * kb + 4 * q4), ve = *(const u32x4*)(el + 32 + 16 * kb + 4 * q4);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          ks[kb][r] = exponent_scale(ke[r]) * a.cx;
          vs[kb][r] = exponent_scale(ve[r]);
        }
      }
    }
    // The next step's rows: as soon as this one's are in registers.  (The share's last step
    // is fetched once more, for no one.)
    const uint32_t here = there;
    there = place(nxt);
    lds_done();
    look_up(then);
    fetch_exps();
    fetch(kl_at, 0);

    // ---- scores: keys 16kb + 4q4 + r, query row 16rb + c16 ----
    f32x4 s[NRB][KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb) s[rb][kb] = f32x4{};
      if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < W / 16; ++j) {
          f32x4 k;
          if constexpr (QUANT) k = codes4(kf[kb][j / 4][j % 4]);
          else k = __builtin_bit_cast(f32x4, kf[kb][j]);
#pragma unroll
          for (int rb = 0; rb < NRB; ++rb)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[rb][kb] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[e], qf[rb][j][e], s[rb][kb], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int j = 0; j < W / 32; ++j) {
          typename E::v8 k;
          if constexpr (QUANT) k = codes8<E>(kf[kb][j / 2][2 * (j % 2)], kf[kb][j / 2][2 * (j % 2) + 1]);
          else k = E::as8(kf[kb][j]);
#pragma unroll
          for (int rb = 0; rb < NRB; ++rb) s[rb][kb] = E::mma16(k, E::as8(qf[rb][j]), s[rb][kb]);
        }
      }
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[rb][kb][r] *= QUANT ? ks[kb][r] : a.cx;
    }
    // Keys that some row does not see: past its own, past the wave's, of missing pages.
    const bool whole = here == (uint32_t)((1ull << KS) - 1) && k0 + KS <= cur.len - (a.T - 1);
    auto sees = [&](int rb, int j) { return (here >> j & 1u) != 0u && k0 + j < lim[rb]; };
    if (!whole) {
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (!sees(rb, 16 * kb + 4 * q4 + r)) s[rb][kb][r] = -INFINITY;
    }

    // ---- online softmax; the running maximum is raised when it is 2^8 behind ----
    float step_scale[NRB];  // of this step's weights
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
      float mx = -INFINITY;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[rb][kb][r]);
      mx = xor32_max(xor16_max(mx));
      if (wave_any(mx > m_run[rb] + kRescaleLog2)) {
        const float m_new = fmaxf(m_run[rb], mx), corr = fast_exp2(m_run[rb] - m_new);
        m_run[rb] = m_new;
        l_run[rb] *= corr;
#pragma unroll
        for (int i = 0; i < NDB; ++i) acc[rb][i] *= corr;
      }
      const float top = STEP_MAX ? fmaxf(mx, kMaxInit) : m_run[rb];
      float rs = 0.f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = fast_exp2(s[rb][kb][r] - top);
          rs += x;
          s[rb][kb][r] = QUANT ? x * vs[kb][r] : x;
        }
      step_scale[rb] = STEP_MAX ? fast_exp2(top - m_run[rb]) : 1.f;
      l_run[rb] = STEP_MAX ? fmaf(rs, step_scale[rb], l_run[rb]) : l_run[rb] + rs;
      if constexpr (QUANT) {
        if (!whole) {  // (what no key was written to may hold 255, an infinite power)
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!sees(rb, 16 * kb + 4 * q4 + r)) s[rb][kb][r] = 0.f;
        }
      }
    }

    // ---- O += P V ----
    arrived<NL + (QUANT ? 2 : 1)>();  // V's rows; behind them the next step's pages, exponents and K
    // V: the operand blocks' rows are dims, their columns the keys 4q4 + j and 16 + 4q4 + j
    // (float32: the rows of four blocks are 4 c16 + i of 64 dims, keys 4q4 + e)
    u32x4 vf[F32 ? KB * NDB : NDB];
    if constexpr (F32) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < NDB / 4; ++i) {
            const int r = 16 * kb + 4 * q4 + e;
            if constexpr (QUANT) vf[kb * NDB + i * 4][e] = *(const uint32_t*)(vl + T::at(r, 4 * i + c16 / 4) + 4 * (c16 & 3));
            else vf[kb * NDB + e * (NDB / 4) + i] = *(const u32x4*)(vl + T::at(r, 16 * i + c16));
          }
    } else if constexpr (QUANT) {
      const int r = (c16 & 8 ? 16 : 0) + 4 * q4 + ((c16 >> 1) & 3);
#pragma unroll
      for (int i = 0; i < NDB; ++i) {
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        const auto x = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (__attribute__((address_space(3))) i32x2*)(vl + T::at(r, i) + 8 * (c16 & 1)));
        vf[i][0] = (uint32_t)x[0];
        vf[i][1] = (uint32_t)x[1];
      }
    } else {
      const int r = 4 * q4 + (c16 >> 2);
#pragma unroll
      for (int i = 0; i < NDB; ++i) {
        const u32x2 lo = lds_read_tr16(vl + T::at(r, 2 * i + ((c16 >> 1) & 1)) + 8 * (c16 & 1));
        const u32x2 hi = lds_read_tr16(vl + T::at(16 + r, 2 * i + ((c16 >> 1) & 1)) + 8 * (c16 & 1));
        vf[i] = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    }

    // An infinity or NaN must not reach the rows that do not see its key.  In the rows that
    // do, the two parts of a 16-bit weight would make a NaN of an infinity (0 or less times
    // it, from the second part), so 16 bits are looked at in every step.
    bool apart = false;
    if constexpr (QUANT) {
      if (!whole) {
        bool odd = false;
#pragma unroll
        for (int i = 0; i < (F32 ? KB * NDB : NDB); ++i) {
          if (F32 && i % 4) continue;  // (four blocks' codes are in the first's dwords)
#pragma unroll
          for (int e = 0; e < (F32 ? 4 : 2); ++e) odd |= odd_codes(vf[i][e]);
        }
        apart = wave_any(odd);
      }
    } else if (!F32 || !whole) {
      apart = wave_any(any_odd<C>(vf));
    }
    if (apart) {
      // one key after the other, for the rows that see it
      const int r16 = once(c16), d4 = once(q4);
#pragma unroll 1
      for (int j = 0; j < KS; ++j) {
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb) {
          float x = 0.f;  // the weight of key j = 16kb + 4qq + r, which lane 16qq + c16 holds
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float y = __shfl(s[rb][kb][r], 16 * ((j >> 2) & 3) + r16);
              x = 16 * kb + r == (j & 19) ? y : x;
            }
          if constexpr (STEP_MAX) x *= step_scale[rb];
          const bool see = sees(rb, j);
#pragma unroll
          for (int i = 0; i < NDB; ++i) {
            f32x4 v;
            if constexpr (F32) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int d = 64 * (i / 4) + 4 * (4 * d4 + e) + i % 4;
                if constexpr (QUANT) v[e] = codes4(vl[T::at(j, d / 16) + d % 16])[0];
                else v[e] = *(const float*)(vl + T::at(j, d / 4) + 4 * (d % 4));
              }
            } else if constexpr (QUANT) {
              v = codes4(*(const uint32_t*)(vl + T::at(j, i) + 4 * d4));
            } else {
              const u32x2 u = *(const u32x2*)(vl + T::at(j, 2 * i + (d4 >> 1)) + 8 * (d4 & 1));
              v = f32x4{C::lo(u[0]), C::hi(u[0]), C::lo(u[1]), C::hi(u[1])};
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (see) acc[rb][i][e] = fmaf(x, v[e], acc[rb][i][e]);
          }
        }
      }
    }
    lds_done();
    fetch(vl_at, 32);
    if (!apart) {
      if constexpr (F32) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < NDB / 4; ++i) {
              f32x4 v;
              if constexpr (QUANT) v = codes4(vf[kb * NDB + i * 4][e]);
              else v = __builtin_bit_cast(f32x4, vf[kb * NDB + e * (NDB / 4) + i]);
#pragma unroll
              for (int rb = 0; rb < NRB; ++rb)
#pragma unroll
                for (int t = 0; t < 4; ++t)
                  acc[rb][4 * i + t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[t], s[rb][kb][e], acc[rb][4 * i + t], 0, 0, 0);
            }
      } else {
        u32x4 pk[NRB], rest[NRB];
#pragma unroll
        for (int rb = 0; rb < NRB; ++rb)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            constexpr float up = STEP_MAX ? kUp : 1.f, rest_up = STEP_MAX ? kRestUp : 1.f;
            const float x = s[rb][i / 2][2 * (i % 2)] * up, y = s[rb][i / 2][2 * (i % 2) + 1] * up;
            pk[rb][i] = EV::pack2(x, y);
            rest[rb][i] = EV::pack2((x - EV::lo(pk[rb][i])) * rest_up, (y - EV::hi(pk[rb][i])) * rest_up);
          }
#pragma unroll
        for (int i = 0; i < NDB; ++i) {
          typename EV::v8 v;
          if constexpr (QUANT) v = codes8<EV>(vf[i][0], vf[i][1]);
          else v = EV::as8(vf[i]);
#pragma unroll
          for (int rb = 0; rb < NRB; ++rb) {
            if constexpr (STEP_MAX) {
              const f32x4 x = EV::mma16(v, EV::as8(pk[rb]), f32x4{}), y = EV::mma16(v, EV::as8(rest[rb]), f32x4{});
              const float xs = step_scale[rb] / kUp, ys = step_scale[rb] / (kUp * kRestUp);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[rb][i][e] = fmaf(x[e], xs, fmaf(y[e], ys, acc[rb][i][e]));
            } else {
              acc[rb][i] = EV::mma16(v, EV::as8(pk[rb]), acc[rb][i]);
              acc[rb][i] = EV::mma16(v, EV::as8(rest[rb]), acc[rb][i]);
            }
          }
        }
      }
    }

    if constexpr (WHOLE) {
      if (cur.left <= 1) break;
    }
    // ---- the end of a sequence, or of the share ----
    if (!WHOLE && (cur.left <= 1 || nxt.b != cur.b)) {
      const bool alone = from_start && k0 + KS >= cur.len;  // the whole sequence
      const int r16 = once(c16), d4 = once(q4);
#pragma unroll
      for (int rb = 0; rb < NRB; ++rb) {
        const int row = row0 + 16 * rb + r16;
        const float den = xor32_sum(xor16_sum(l_run[rb]));
        if (row >= a.rows) continue;
        const bool some = bits_of(den) != 0u;
        const float inv = some ? 1.f / den : 0.f;
        const int gi = a.by_t(row), t = row - gi * a.T, hq = g * (a.Hq / p.H) + gi;
        const int64_t at = alone ? ((int64_t)cur.b * a.T + t) * a.Hq + hq : ((int64_t)(share + cur.b) * p.H + g) * a.rows + row;
#pragma unroll
        for (int i = 0; i < NDB; ++i) {
          f32x4 x = acc[rb][i];
          int d = 16 * i + 4 * d4;
          if constexpr (F32) {  // dims 64j + 16q4 + 4r ..: element r of the four blocks 4j ..
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] = acc[rb][i / 4 * 4 + u][i % 4];
            d = 64 * (i / 4) + 16 * d4 + 4 * (i % 4);
          }
          if (ROWS && d >= a.D) continue;
          if (alone) {
#pragma unroll
            for (int u = 0; u < 4; ++u) x[u] *= inv;
            char* to = a.o + (at * a.D + d) * ES;
            if constexpr (F32) *(f32x4*)to = x;
            else *(u32x2*)to = u32x2{E::pack2(x[0], x[1]), E::pack2(x[2], x[3])};
          } else {
            *(f32x4*)(a.ws_o + at * W + d) = x;
          }
        }
        if (d4 == 0) {
          if (!alone) *(float2*)(a.ws_ml + 2 * at) = make_float2(m_run[rb], den);
          else if (a.lse) a.lse[((int64_t)cur.b * a.Hq + hq) * a.T + t] = some ? (m_run[rb] + __log2f(den)) * kLn2 : INFINITY;
        }
      }
      if (cur.left <= 1) break;
      begin(nxt);
    }
    cur = nxt;
    nxt = then;
    then = next_step(a, lens, then);
  }
  arrived<0>();  // (nothing may come to LDS that is another's by then)

  if constexpr (WHOLE) {
    // ---- the waves' (max, sum, O), one block of rows at a time; the first half of the dims
    // through K's memory, the second through V's: quad c of row r at c ^ r ----
    constexpr int NQ = W / 4, HQ = NQ / 2;  // quads of dims of a row, and of a half
#pragma unroll
    for (int rb = 0; rb < NRB; ++rb) {
      const float l = xor32_sum(xor16_sum(l_run[rb]));
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NDB; ++i) {
        f32x4 x = acc[rb][i];
        int quad = 4 * i + q4;
        if constexpr (F32) {  // quad 16j + 4q4 + r: element r of the four blocks 4j ..
#pragma unroll
          for (int u = 0; u < 4; ++u) x[u] = acc[rb][i / 4 * 4 + u][i % 4];
          quad = i / 4 * 16 + 4 * q4 + i % 4;
        }
        unsigned char* to = quad < HQ ? k_lds : v_lds;
        *(f32x4*)(to + ((w * 16 + c16) * HQ + ((quad % HQ) ^ (c16 & (HQ - 1)))) * 16) = x;
      }
      if (q4 == 0) ml_lds[w * 16 + c16] = make_float2(m_run[rb], l);
      __syncthreads();
      const int nr = min(16, a.rows - row0 - 16 * rb);
      for (int e = threadIdx.x; e < nr * NQ; e += 64 * NW) {
        const int r = e / NQ, c = e % NQ;
        if (ROWS && 4 * c >= a.D) continue;
        float M = kMaxInit, den = 0.f;
#pragma unroll
        for (int x = 0; x < NW; ++x) M = fmaxf(M, ml_lds[x * 16 + r].x);
        f32x4 O = {};
        const unsigned char* from = c < HQ ? k_lds : v_lds;
#pragma unroll
        for (int x = 0; x < NW; ++x) {
          const float2 ml = ml_lds[x * 16 + r];
          const float f = fast_exp2(ml.x - M);
          den = fmaf(f, ml.y, den);
          const f32x4 o = *(const f32x4*)(from + ((x * 16 + r) * HQ + ((c % HQ) ^ (r & (HQ - 1)))) * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) O[i] = fmaf(f, o[i], O[i]);
        }
        const int row = row0 + 16 * rb + r, gi = a.by_t(row), t = row - gi * a.T, hq = g * (a.Hq / p.H) + gi;
        const bool some = bits_of(den) != 0u;
        const float inv = some ? 1.f / den : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) O[i] *= inv;
        char* to = a.o + ((((int64_t)cur.b * a.T + t) * a.Hq + hq) * a.D + 4 * c) * ES;
        if constexpr (F32) *(f32x4*)to = O;
        else *(u32x2*)to = u32x2{E::pack2(O[0], O[1]), E::pack2(O[2], O[3])};
        if (a.lse && c == 0) a.lse[((int64_t)cur.b * a.Hq + hq) * a.T + t] = some ? (M + __log2f(den)) * kLn2 : INFINITY;
      }
    }
  }
}

// Joins the parts of a sequence: 256 >> a.slices quads of dims of a (sequence, KV head) to
// a workgroup, 1 << a.slices threads to a quad, which take every so manieth part, 8 of a
// thread in flight.  Sequences of one part are finished; those without keys give 0 and LSE
// +inf.
template <typename E, int W>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  constexpr int NQ = W / 4, U = 8;
  __shared__ f32x4 o_lds[256];
  __shared__ float2 ml_lds[256];
  const int tid = threadIdx.x, per = 256 >> a.slices, sl = tid >> (8 - a.slices), step = 1 << a.slices;
  const int quad = blockIdx.x * per + (tid & (per - 1)), row = quad / NQ, c = quad % NQ;
  const bool in = row < a.rows && 4 * c < a.D;
  const Lane all = lane_steps(a);
  const int size = share_of(a, all_steps(a, all));
  for (int pair = blockIdx.y; pair < a.B * a.p.H; pair += gridDim.y) {
    const int b = a.by_g(pair), g = pair - b * a.p.H;
    int steps;
    const int from = steps_before(a, all, b, steps), share = from / size;
    const int n = steps ? (from + steps - 1) / size - share + 1 : 0;
    if (n == 1) continue;
    float M = kMaxInit, den = 0.f;
    f32x4 O = {};
    const int64_t first = ((int64_t)(share + b) * a.p.H + g) * a.rows + (in ? row : 0), apart = (int64_t)a.p.H * a.rows;
    for (int x0 = sl; x0 < n; x0 += U * step) {
      float2 ml[U];
      f32x4 o[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool ok = in && x0 + u * step < n;
        const int64_t at = first + (ok ? x0 + u * step : x0) * apart;
        ml[u] = ok ? *(const float2*)(a.ws_ml + 2 * at) : make_float2(kMaxInit, 0.f);
        o[u] = ok ? *(const f32x4*)(a.ws_o + at * W + 4 * c) : f32x4{};
      }
      float m = M;
#pragma unroll
      for (int u = 0; u < U; ++u) m = fmaxf(m, ml[u].x);
      const float f = fast_exp2(M - m);
      M = m;
      den *= f;
      O *= f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float y = fast_exp2(ml[u].x - M);
        den = fmaf(y, ml[u].y, den);
#pragma unroll
        for (int i = 0; i < 4; ++i) O[i] = fmaf(y, o[u][i], O[i]);
      }
    }
    if (a.slices) {
      __syncthreads();  // (the pair before is done with the memory)
      ml_lds[tid] = make_float2(M, den);
      o_lds[tid] = O;
      __syncthreads();
      if (sl) continue;
      for (int x = 1; x < step; ++x) M = fmaxf(M, ml_lds[tid + x * per].x);
      den = 0.f;
      O = f32x4{};
      for (int x = 0; x < step; ++x) {
        const float2 ml = ml_lds[tid + x * per];
        const f32x4 o = o_lds[tid + x * per];
        const float y = fast_exp2(ml.x - M);
        den = fmaf(y, ml.y, den);
#pragma unroll
        for (int i = 0; i < 4; ++i) O[i] = fmaf(y, o[i], O[i]);
      }
    }
    if (!in) continue;
    const int gi = a.by_t(row), t = row - gi * a.T, hq = g * (a.Hq / a.p.H) + gi;
    const bool some = bits_of(den) != 0u;
    f32x4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = some ? O[i] / den : 0.f;
    char* to = a.o + ((((int64_t)b * a.T + t) * a.Hq + hq) * a.D + 4 * c) * fmt_size<E>();
    if constexpr (std::is_same<E, F32Fmt>::value) *(f32x4*)to = out;
    else *(u32x2*)to = u32x2{E::pack2(out[0], out[1]), E::pack2(out[2], out[3])};
    if (a.lse && c == 0) a.lse[((int64_t)b * a.Hq + hq) * a.T + t] = some ? (M + __log2f(den)) * kLn2 : INFINITY;
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
static int paged_width(int64_t head_dim) { return head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256; }
// Blocks of 16 query rows of a wave: 32 rows of 256 features spill registers.
static int paged_blocks(int64_t rows, int64_t head_dim) { return rows > 16 && paged_width(head_dim) < 256 ? 2 : 1; }
static int64_t paged_groups(int64_t rows, int64_t head_dim) {
  const int64_t n = 16 * paged_blocks(rows, head_dim);
  return std::max<int64_t>((rows + n - 1) / n, 1);
}
// Shares of a KV head, with `waves` waves to a compute unit at a time: as many as fill the
// device once, each of the groups of rows taking all of them.
static int64_t paged_shares(int64_t kv_heads, int64_t rows, int64_t head_dim, int waves) {
  return std::max<int64_t>((int64_t)256 * waves / (kv_heads * paged_groups(rows, head_dim)), 1);
}
// Parts of a KV head at most: one of every share, and one more where a sequence begins.
static int64_t paged_parts(int64_t batch, int64_t kv_heads, int64_t rows, int64_t head_dim) {
  return paged_shares(kv_heads, rows, head_dim, kPagedWaves) + batch;
}
static size_t paged_ws(int64_t batch, int64_t kv_heads, int64_t rows, int64_t head_dim) {
  return (size_t)(paged_parts(batch, kv_heads, rows, head_dim) * kv_heads * rows * (paged_width(head_dim) + 2)) * sizeof(float) + 16;
}
static_assert(paged_waves<Bf16Fmt, 64>() <= kPagedWaves && paged_waves<E4m3Fmt, 64>() <= kPagedWaves,
              "paged_parts counts the shares of so many waves");

// Whether a workgroup takes a sequence whole, and nothing is joined after it: where one
// compute unit has little enough to read (by itself it reads some 40 GB/s).  us in a
// captured graph, whole / shares and join, 1, 8 and 32 sequences, 8 KV heads:
//                        128 KB and less               256 KB
//   bf16, 128 features   256 keys  6.3 / 8.9           512 keys  7.7 / 9.1
//                                  6.9 / 10.3                    11.4 / 10.7
//                                  9.1 / 12.1                    15.2 / 15.6
//   8 bits, the same     512 keys  7.2 / 9.2           1024 keys 10.1 / 9.6
//                                  7.6 / 10.5                    10.5 / 11.4
//                                  9.2 / 14.6                    16.2 / 19.6
//   bf16, 64 features    512 keys  5.7 / 8.1           1024 keys 7.8 / 8.3
//                                  6.3 / 9.3                     11.9 / 9.9
//                                  8.5 / 11.7                    14.5 / 15.8
//   float32, 64          256 keys  7.8 / 8.4           512 keys  11.2 / 8.7
//                                  8.5 / 9.2                     12.2 / 9.9
//                                  10.7 / 12.6                   16.1 / 16.5
// Up to 128 KB whole is faster at any number of sequences.  At 256 KB either side can be;
// which one depends on the number of workgroups too, and the shares taken there cost up to
// 1.4 us with one sequence and 3.4 with 32.
constexpr int64_t kWholeBytes = 128 << 10;
static bool paged_whole(int64_t capacity, int64_t row_bytes) { return capacity * 2 * row_bytes <= kWholeBytes; }

template <typename C, typename E, int W, bool ROWS>
static int run_paged(PagedArgs& a, hipStream_t s, const char* who) {
  constexpr int NRB = W == 256 ? 1 : 2;
  const bool two = paged_blocks(a.rows, W) == 2;
  a.step_log = PageTile<C, W>::KS == 16 ? 4 : 5;
  const int64_t capacity = (int64_t)a.p.most * a.p.page;
  const unsigned groups = (unsigned)paged_groups(a.rows, W);
  if (paged_whole(capacity, PageTile<C, W>::ROWB)) {
    const dim3 grid((unsigned)(a.B * a.p.H), groups);
    if (two) launch_kernel<paged_decode_kernel<C, E, W, NRB, ROWS, true>>(grid, dim3(64 * paged_whole_waves<C, E, W, NRB>()), 0, s, a);
    else launch_kernel<paged_decode_kernel<C, E, W, 1, ROWS, true>>(grid, dim3(64 * paged_whole_waves<C, E, W, 1>()), 0, s, a);
    return check_launch(who);
  }
  a.shares = (int)paged_shares(a.p.H, a.rows, W, paged_waves<C, W>());
  a.by_shares = fast_div(a.shares);
  a.least = least_share<E>() >> a.step_log;
  const int64_t steps = a.B * ((capacity + PageTile<C, W>::KS - 1) >> a.step_log);
  if (a.shares > (steps + a.least - 1) / a.least) a.shares = (int)((steps + a.least - 1) / a.least), a.by_shares = fast_div(a.shares);
  const int group = paged_group<C, W>(), gx = (a.shares * a.p.H + group - 1) / group;
  const dim3 grid((unsigned)gx, groups);
  if (two) launch_kernel<paged_decode_kernel<C, E, W, NRB, ROWS, false>>(grid, dim3(64 * group), 0, s, a);
  else launch_kernel<paged_decode_kernel<C, E, W, 1, ROWS, false>>(grid, dim3(64 * group), 0, s, a);
  int rc = check_launch(who);
  if (rc) return rc;
  // Sequences of more than one part, or of none.  Threads enough that each takes up to 8
  // parts of an even cut (131072 keys of one sequence, 255 parts: 5.1 us against 9.5 with a
  // workgroup to a row), and that the rows fill a workgroup.
  const int64_t quads = (int64_t)a.rows * (W / 4), parts = a.shares / a.B + 1;
  while (a.slices < 5 && (parts > 8 << a.slices || quads << a.slices < 256)) ++a.slices;
  const int per = 256 >> a.slices;
  launch_kernel<paged_join_kernel<E, W>>(dim3((unsigned)((quads + per - 1) / per), (unsigned)std::min(a.B * a.p.H, 65535)),
                                         dim3(256), 0, s, a);
  return check_launch(who);
}
template <typename C, typename E, int W>
static int run_paged(PagedArgs& a, hipStream_t s, const char* who) {
  return a.D < W ? run_paged<C, E, W, true>(a, s, who) : run_paged<C, E, W, false>(a, s, who);
}
template <typename C, typename E>
static int run_paged(PagedArgs& a, hipStream_t s, const char* who) {
  const int w = paged_width(a.D);
  return w == 64 ? run_paged<C, E, 64>(a, s, who) : w == 128 ? run_paged<C, E, 128>(a, s, who) : run_paged<C, E, 256>(a, s, who);
}

}  // namespace pjx

using namespace pjx;

extern "C" size_t pjx_paged_decode_workspace_size(int64_t batch, int64_t kv_heads, int64_t rows, int64_t capacity,
                                                  int64_t head_dim) {
  if (batch < 0 || kv_heads <= 0 || rows < 0 || capacity < 0) return 16;
  return paged_ws(batch, kv_heads, rows, head_dim);
}

extern "C" int pjx_paged_decode(int dtype, int cache_dtype, const void* q, const pjx_pages* cache,
                                const int32_t* kv_lengths, void* o, float* lse, void* workspace,
                                size_t workspace_bytes, int64_t batch, int64_t q_len, int64_t q_heads,
                                int64_t kv_heads, int64_t head_dim, float sm_scale, void* stream) {
  clear_error();
  const char* who = "pjx_paged_decode";
  PagedArgs a = {};
  const int rc = fill_pages(a.p, who, cache_dtype, cache, batch, kv_heads, head_dim);
  if (rc != PJX_OK) return rc;
  if (dtype != PJX_DTYPE_BF16 && dtype != PJX_DTYPE_F16 && dtype != PJX_DTYPE_F32)
    return fail(PJX_ERR_INVALID, "pjx_paged_decode: dtype must be PJX_DTYPE_BF16, PJX_DTYPE_F16 or PJX_DTYPE_F32");
  const bool quant = cache_dtype == PJX_DTYPE_E4M3, f32 = dtype == PJX_DTYPE_F32;
  if (!quant && cache_dtype != dtype) return fail(PJX_ERR_INVALID, "pjx_paged_decode: the cache has another dtype");
  if (q_len <= 0 || q_heads <= 0 || q_heads % kv_heads) return fail(PJX_ERR_INVALID, "pjx_paged_decode: bad sizes");
  const int64_t rows = q_heads / kv_heads * q_len, capacity = cache->page_size * cache->table_len;
  if (q_len > (1 << 20) || q_heads > (1 << 20) || rows > (1 << 19) || batch * kv_heads > (1 << 22) ||
      batch * kv_heads * rows > (1 << 30))
    return fail(PJX_ERR_INVALID, "pjx_paged_decode: sizes out of range");
  if (batch * ((capacity + 15) / 16) > (1 << 30))
    return fail(PJX_ERR_INVALID, "pjx_paged_decode: the sequences have room for more than 2^34 keys");
  if (!(sm_scale > 0.f)) return fail(PJX_ERR_INVALID, "pjx_paged_decode: sm_scale must be > 0");
  if (batch == 0) return PJX_OK;
  if (!q || !o) return fail(PJX_ERR_INVALID, "pjx_paged_decode: null pointer");
  if (((uintptr_t)q | (uintptr_t)o) % 16) return fail(PJX_ERR_INVALID, "pjx_paged_decode: q and o must start on 16 bytes");
  hipStream_t s = (hipStream_t)stream;
  if (capacity == 0 || cache->pages == 0)
    return write_keyless(o, lse, (size_t)(batch * q_len * q_heads * head_dim), f32, (size_t)(batch * q_heads * q_len), s,
                         who);
  if (!workspace || workspace_bytes < paged_ws(batch, kv_heads, rows, head_dim))
    return fail(PJX_ERR_WORKSPACE, "pjx_paged_decode: workspace missing or too small");
  if ((uintptr_t)workspace % 16) return fail(PJX_ERR_INVALID, "pjx_paged_decode: the workspace must start on 16 bytes");
  a.q = (const char*)q; a.o = (char*)o; a.lse = lse; a.lengths = kv_lengths;
  a.B = (int)batch; a.T = (int)q_len; a.Hq = (int)q_heads; a.D = (int)head_dim; a.rows = (int)rows;
  a.by_g = fast_div(kv_heads);
  a.by_t = fast_div(q_len);
  a.cx = sm_scale * kLog2e;
  a.ws_o = (float*)workspace;
  a.ws_ml = a.ws_o + paged_parts(batch, kv_heads, rows, head_dim) * kv_heads * rows * paged_width(head_dim);
  if (f32) return quant ? run_paged<E4m3Fmt, F32Fmt>(a, s, who) : run_paged<F32Fmt, F32Fmt>(a, s, who);
  if (dtype == PJX_DTYPE_BF16) return quant ? run_paged<E4m3Fmt, Bf16Fmt>(a, s, who) : run_paged<Bf16Fmt, Bf16Fmt>(a, s, who);
  return quant ? run_paged<E4m3Fmt, F16Fmt>(a, s, who) : run_paged<F16Fmt, F16Fmt>(a, s, who);
}
