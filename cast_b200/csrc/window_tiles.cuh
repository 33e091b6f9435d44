// Sliding-window attention for many query rows: tcgen05 products with TMEM
// accumulators over the keys that the rows of a tile see.
//
// The mathematics and the list of keys are those of window.cuh.  One CTA
// computes one 128-row query tile, and two CTAs (heads of 64: four) share an
// SM: the start and end of one overlap the steps of the others, which a short
// window has few of (two tiles a CTA on one key list took 212 us for the prompt
// below).  The
// `pack` query heads that share a key head lie side by side in the rows (row =
// token * pack + head), so a tile covers 128 / pack tokens and their windows
// differ by little.  Keys go by in tiles of 64 places of the list (8-row
// aligned, so that the sinks' last rows and the window's first ones share a
// tile: two TMA boxes).  Step h is one key tile:
//   S(h) = Q K_h^T       tcgen05, f32 in a 64-column TMEM buffer (one of two)
//   P(h) = 2^(S c - m)   one softmax thread a row, written over S(h) in pairs
//   O   += P(h) V_h      tcgen05, A = P from TMEM
// with the lazily moved maximum and the single pass of attention.cuh.
//   warps 0-3  softmax and epilogue (TMEM lanes 0..127)
//   warp 4     TMA of Q and the K ring      warp 5  MMA issuer (one thread)
//   warp 6     TMA of the V ring            warp 7  idle
//
// Masks cost only where they are: a warp whose 32 rows all see a step's keys
// runs the unmasked step, and one that sees none of them writes zeros without
// an exponential.  A V row meets the zero weights of rows that do not see it,
// and 0 * inf is NaN, so warp 6 goes over the V tiles that are not wholly
// visible before they are used: rows that nobody sees become zeros; in rows
// that only some see, infinities and NaN become zeros and are given back to
// the rows that see them when these are written.
//
// Bound: the softmax warps' steps.  Measured (bf16, heads of 128, in a graph;
// in brackets calls one after the other): 24 heads of 3520 queries over 9
// frames of 880, 311 to 337 us (365: the power cap) = 1.10 PFLOP/s of visible
// pairs, 0.68 of the measured bf16 peak (exponentials 0.57 of their pipe, tensor
// pipe 0.55); 32 / 8 heads, 8192 queries, window 1024, 4 sinks: 155 us (174), of
// which about a quarter is the start and end of items of 18 steps.  Heads of 64
// are bound by one S buffer a CTA, whose step is one chain: fp16, 16 / 4 heads,
// 3 x 1001 queries over 777 keys, 29 us (30), 384 items on 592 places in one wave
// (exponentials 0.38 of their pipe, tensor pipe 0.15).
#pragma once

#include "window.cuh"

namespace castk {

constexpr int kTilesThreads = 256;
constexpr int kTilesPartCols = 4;  // m, l, flag (and nothing) of a part's rows beside its O

// What depends on the head vectors' length.  128: TMEM holds O (128 columns)
// and two S buffers for two CTAs, so that S of the next step is there while the
// softmax works.  64: O takes half, and four CTAs with one S buffer each keep
// the exponentials busier than two with two (twice the softmax warps).
template <int D>
struct TilesSmem {
  static constexpr int ctas = D == 128 ? 2 : 4;    // on an SM
  static constexpr int bufs = D == 128 ? 2 : 1;    // S buffers
  static constexpr int chunk = D == 128 ? 64 : 32; // scores a thread holds at a time
  // Registers of a thread of the softmax warps and of the others; their sum
  // times 128 is the block's share of the SM at launch, 65536 / ctas.
  static constexpr int regs_soft = D == 128 ? 200 : 88, regs_rest = D == 128 ? 56 : 40;
  static constexpr int tmem_cols = D == 128 ? 256 : 128, s_col = D;  // O in columns [0, D)
  static constexpr int keys = 64;  // of one K or V tile: one step
  static constexpr int q_tile = 128 * D * 2;
  static constexpr int tile = keys * D * 2;
  static constexpr int half = keys * 128;  // 64 columns of a tile
  static constexpr int stages = 2;
  static constexpr int k_off = q_tile;
  static constexpr int v_off = k_off + stages * tile;
  static constexpr int bars = v_off + stages * tile;
  // q_full, then [2] each: k_full, v_full, v_raw, s_full, p_full, pv_done, k_free, v_free; drain
  static constexpr int n_bars = 1 + 8 * 2 + 1;
  static constexpr int tmem_slot = bars + 8 * n_bars;
  static constexpr int alloc = tmem_slot + 16;
  static __device__ __forceinline__ int buf(int h) { return bufs == 2 ? h & 1 : 0; }
  static __device__ __forceinline__ uint32_t phase(int h) { return bufs == 2 ? (h >> 1) & 1 : h & 1; }
};

template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

struct TilesParams {
  void *out;
  const void *v;
  long long os[3], vs[3];
  const int32_t *kv_lens;
  float *part;
  WindowRule rule;
  int Lq, lk;
  int pack, pack_log2;   // heads side by side in the rows of a tile, a power of two
  int head_groups;       // Hq / pack
  int groups_per_key;    // head groups that share a key head
  int rows, q_tiles;     // rows = pack * Lq of one head group
  int n_whole, parts;    // items [0, n_whole) whole, the later ones in `parts` parts each
  FastDiv by_tiles, by_groups, by_keys;  // q_tiles, head_groups, groups_per_key
  int sinks8;            // sinks of a session long enough to have a gap, rounded up to 8
  int k_batch, k_head, v_batch, v_head;  // 0 where that dimension's stride is 0 (one box for all), else 1
  float scale_log2;
};

// A part's result: O [column][row], then [m, l, flag][row].
template <int D>
__host__ __device__ constexpr long long tiles_part_floats() {
  return 128ll * (D + kTilesPartCols);
}

template <typename T>
struct TilesType;
template <>
struct TilesType<__nv_bfloat16> {
  static constexpr uint32_t fmt = 1;
  static constexpr float kShift = 0.0f, kSlack = 8.0f, kSumLimit = 65536.0f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  static __device__ __forceinline__ float add_lo(uint32_t u, float x) { return add_bf16_lo(u, x); }
  static __device__ __forceinline__ float add_hi(uint32_t u, float x) { return add_bf16_hi(u, x); }
};
template <>
struct TilesType<__half> {
  // P = 2^(s - m + 8): none is above 2^12 without a move of the maximum (a chunk
  // of P that sums to more than 2^15 is looked at again), and weights down to
  // 2^-32 of the largest count
  static constexpr uint32_t fmt = 0;
  static constexpr float kShift = 8.0f, kSlack = 4.0f, kSumLimit = 32768.0f;
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return Half2<__half>::pack(a, b); }
  static __device__ __forceinline__ float add_lo(uint32_t u, float x) {
    float r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tadd.rn.f32.f16 %0, lo, %2;\n\t}" : "=f"(r) : "r"(u), "f"(x));
    return r;
  }
  static __device__ __forceinline__ float add_hi(uint32_t u, float x) {
    float r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tadd.rn.f32.f16 %0, hi, %2;\n\t}" : "=f"(r) : "r"(u), "f"(x));
    return r;
  }
};

__device__ __forceinline__ void tma_load_5d(void *dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1, int c2,
                                            int c3, int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(castdev::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(castdev::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}

__device__ __forceinline__ void tma_store_5d(const CUtensorMap *map, const void *src, int c0, int c1, int c2, int c3,
                                             int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4, %5, %6}], [%1];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(castdev::smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}

// Bits n0 .. n0+31 of the interval [lo, hi).
__device__ __forceinline__ uint32_t interval_mask(int lo, int hi, int n0) {
  const int a = min(max(lo - n0, 0), 32), b = min(max(hi - n0, 0), 32);
  const uint32_t below_b = b >= 32 ? 0xffffffffu : (1u << b) - 1u;
  const uint32_t below_a = a >= 32 ? 0xffffffffu : (1u << a) - 1u;
  return below_b & ~below_a;
}

// N columns from TMEM into x, there when this returns (x is tied to the wait,
// so that nothing reads it before).
template <int N>
__device__ __forceinline__ void tmem_get(uint32_t addr, uint32_t (&x)[N]) {
  if constexpr (N == 16) {
    castdev::tmem_ld16(addr, x);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 32) castdev::tmem_ld32(addr + i, *reinterpret_cast<uint32_t(*)[32]>(&x[i]));
  }
  castdev::tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(x[i]));
}
__device__ __forceinline__ void tmem_put(uint32_t addr, const uint32_t (&r)[32]) { castdev::tmem_st32(addr, r); }
__device__ __forceinline__ void tmem_put(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// P = 2^(x c2 - base) of N scores in pairs; returns their sum as rounded.
// (Taking an eighth to a half of the exponentials to the FMA pipe with a
// polynomial of degree 3 was slower: 321 to 340 us against 313 for 24 heads of
// 3520 queries over 7920 keys; it takes ten issue slots for each.)
template <typename T, bool kMasked, int N>
__device__ __forceinline__ float tiles_probs(const uint32_t (&x)[N], uint32_t (&pk)[N / 2], const uint32_t (&seen)[N / 32],
                                             float c2, float base) {
  using X = TilesType<T>;
  const uint64_t c2x2 = f2_pack(c2, c2), nbx2 = f2_pack(-base, -base);
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < N / 2; ++c) {
    float x0, x1;
    f2_unpack(f2_fma(f2_pack(__uint_as_float(x[2 * c]), __uint_as_float(x[2 * c + 1])), c2x2, nbx2), x0, x1);
    float e0 = fast_exp2(x0), e1 = fast_exp2(x1);
    if (kMasked) {
      const uint32_t w = seen[c / 16];
      e0 = ((w >> ((2 * c) % 32)) & 1u) ? e0 : 0.0f;
      e1 = ((w >> ((2 * c + 1) % 32)) & 1u) ? e1 : 0.0f;
    }
    pk[c] = X::pack(e0, e1);
    acc[2 * (c & 3)] = X::add_lo(pk[c], acc[2 * (c & 3)]);
    acc[2 * (c & 3) + 1] = X::add_hi(pk[c], acc[2 * (c & 3) + 1]);
  }
  return ((acc[0] + acc[1]) + (acc[2] + acc[3])) + ((acc[4] + acc[5]) + (acc[6] + acc[7]));
}

// Maximum of the scores that are seen, times c2; -inf where none is.
__device__ __forceinline__ float tiles_max(const uint32_t (&x)[32], uint32_t seen, float c2) {
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < 32; ++c) m[c & 3] = fmaxf(m[c & 3], ((seen >> c) & 1u) ? __uint_as_float(x[c]) : -INFINITY);
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * c2;
}

// Issues the products of one query tile over n 64-key steps.  The S that takes
// the buffer of P of step h (step h + bufs) comes right after P V of step h.
// What can be waited for ahead is, so that only P stands between the softmax
// and the tensor core.  A stage of the K ring is free when its S is done and
// one of the V ring when its P V is: with two S buffers s_full and pv_done say
// so, with one (whose phase may have moved on twice) barriers of their own.
template <typename T, int D>
__device__ __forceinline__ bool tiles_issuer(uint32_t tmem, uint32_t sbase, int n, uint64_t *q_full, uint64_t *k_full,
                                             uint64_t *v_full, uint64_t *s_full, uint64_t *p_full, uint64_t *pv_done,
                                             uint64_t *k_free, uint64_t *v_free, int *err) {
  using S = TilesSmem<D>;
  constexpr uint32_t fmt = TilesType<T>::fmt;
  constexpr uint32_t idesc_s = castdev::make_idesc(1, fmt, fmt, 0, 0, 128, 64);
  constexpr uint32_t idesc_pv = castdev::make_idesc(1, fmt, fmt, 0, 1, 128, D);
  const DescW qd = desc_words(sbase, 16);
  const DescW kd = desc_words(sbase + S::k_off, 16);
  const DescW vd = desc_words(sbase + S::v_off, S::half);
  const uint32_t s_col = tmem + S::s_col;
  auto issue_s = [&](int h) {
    const uint32_t d = s_col + S::buf(h) * 64, ko = (h & 1) * S::tile;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
      castdev::mma_f16_ss(d, qd.at((s >> 2) * 16384 + (s & 3) * 32), kd.at(ko + (s >> 2) * S::half + (s & 3) * 32),
                          idesc_s, s > 0);
    castdev::tc_commit(&s_full[S::buf(h)]);
    if (S::bufs == 1) castdev::tc_commit(&k_free[h & 1]);
  };
  if (!castdev::mbar_wait(q_full, 0, err)) return false;
  for (int h = 0; h < min(n, S::bufs); ++h) {
    if (!castdev::mbar_wait(&k_full[h], 0, err)) return false;
    castdev::tc_fence_after();
    issue_s(h);
  }
  for (int h = 0; h < n; ++h) {
    const int stage = h & 1, next = h + S::bufs;
    const bool more = next < n;
    if (!castdev::mbar_wait(&v_full[stage], (h >> 1) & 1, err)) return false;
    if (more && !castdev::mbar_wait(&k_full[next & 1], (next >> 1) & 1, err)) return false;
    if (!castdev::mbar_wait(&p_full[S::buf(h)], S::phase(h), err)) return false;
    castdev::tc_fence_after();
    const uint32_t vo = stage * S::tile, pa = s_col + S::buf(h) * 64;
#pragma unroll
    for (int s = 0; s < 4; ++s) castdev::mma_f16_ts(tmem, pa + 8 * s, vd.at(vo + 2048 * s), idesc_pv, (h | s) != 0);
    castdev::tc_commit(&pv_done[S::buf(h)]);
    if (S::bufs == 1) castdev::tc_commit(&v_free[stage]);
    if (more) issue_s(next);
  }
  return true;
}

// Gives a row the infinities and NaN of the values that it sees and not every
// row of its item does (columns c0 .. c0 + N - 1); they were taken out of the
// V tiles.  Far off the usual path: a loop over the item's keys.
template <typename T, int N>
__device__ __noinline__ void tiles_give_back(const TilesParams &p, const WindowSpan &span, int b, int hk, int lo, int hi,
                                             int c0, float (&y)[N]) {
  if (hi == 0) return;
  const T *v = static_cast<const T *>(p.v) + b * p.vs[0] + hk * p.vs[1] + c0;
  for (int n = 0; n < span.n; ++n) {
    const int key = span.key(n);
    if (!span.some(key) || !window_sees(key, lo, hi, span.sinks)) continue;
    for (int c = 0; c < N; ++c) {
      const float u = (float)v[key * p.vs[2] + c];
      if (!isfinite(u)) y[c] += u;
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kTilesThreads, TilesSmem<D>::ctas)
    window_tiles_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_k_sink,
                        const __grid_constant__ CUtensorMap tm_v_sink, const __grid_constant__ CUtensorMap tm_k_rest,
                        const __grid_constant__ CUtensorMap tm_v_rest, const __grid_constant__ CUtensorMap tm_o,
                        const __grid_constant__ TilesParams p) {
  using S = TilesSmem<D>;
  using X = TilesType<T>;
  constexpr int KT = S::keys;
  extern __shared__ __align__(1024) uint8_t smem_tiles[];
  uint8_t *smem = smem_tiles;
  uint64_t *bar = reinterpret_cast<uint64_t *>(smem + S::bars);
  uint64_t *q_full = bar;
  uint64_t *k_full = bar + 1;
  uint64_t *v_full = k_full + 2;
  uint64_t *v_raw = v_full + 2;  // a V tile has landed and is gone over before v_full
  uint64_t *s_full = v_raw + 2;
  uint64_t *p_full = s_full + 2;
  uint64_t *pv_done = p_full + 2;
  uint64_t *k_free = S::bufs == 2 ? s_full : pv_done + 2;   // see tiles_issuer
  uint64_t *v_free = S::bufs == 2 ? pv_done : pv_done + 4;
  uint64_t *mma_drain = pv_done + 6;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + S::tmem_slot);
  volatile uint32_t *bad_flag = tmem_slot + 1;  // an infinity or NaN was taken out of a V tile
  int *err = reinterpret_cast<int *>(tmem_slot + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- the item, and which part of its key tiles
  int x = blockIdx.x, part = 0, n_parts = 1;
  if (x >= p.n_whole) {
    part = (x - p.n_whole) % p.parts;
    x = p.n_whole + (x - p.n_whole) / p.parts;
    n_parts = p.parts;
  }
  const int bhg = p.by_tiles.div(x);
  const int qt = p.q_tiles - 1 - (x - bhg * p.q_tiles);  // later rows see more keys: first
  const int b = p.by_groups.div(bhg), hg = bhg - b * p.head_groups;
  const int hk = p.by_keys.div(hg);
  const int row0 = qt * 128, row_end = min(p.rows, row0 + 128);
  int len = p.kv_lens ? p.kv_lens[b] : p.lk;
  if (len < 0 || len > p.lk) {  // a session longer than its keys: nothing past them is read
    if (threadIdx.x == 0) atomicExch(&g_cast_device_error, (int)CAST_ERR_INVALID_ARGUMENT);
    len = min(max(len, 0), p.lk);
  }
  const WindowSpan span = window_span(p.rule, len, p.Lq, row0 >> p.pack_log2, (row_end - 1) >> p.pack_log2);
  // places: [0, s_n) sinks, [s_n, s8) nothing, from s8 the keys from span.base on
  const int s8 = span.s_n > 0 ? p.sinks8 : 0;
  const int n_places = span.n - span.s_n + s8;
  const int n_tiles = span.n > 0 ? (n_places + KT - 1) / KT : 0;
  int kt_lo = 0, n_kv = n_tiles;
  if (n_parts > 1) {  // an equal share, the first parts one more
    const int share = n_tiles / n_parts, more = n_tiles - share * n_parts;
    kt_lo = part * share + min(part, more);
    n_kv = share + (part < more ? 1 : 0);
  }
  constexpr int kKWarp = 4, kMWarp = 5, kVWarp = 6;

  // Starts the copies of the tile of KT places from place n0 on.
  auto start = [&](uint8_t *dst, uint64_t *full, int n0, const CUtensorMap *whole, const CUtensorMap *sink,
                   const CUtensorMap *rest, int head, int batch) {
    if (n0 >= s8 || n0 + KT <= s8) {
      const int key = n0 >= s8 ? span.base + n0 - s8 : n0;
#pragma unroll
      for (int h = 0; h < D / 64; ++h) castdev::tma_load_4d(dst + h * S::half, whole, full, 64 * h, key, head, batch);
    } else {
      const int r = s8 - n0;
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        castdev::tma_load_4d(dst + h * S::half, sink, full, 64 * h, n0, head, batch);
        castdev::tma_load_4d(dst + h * S::half + r * 128, rest, full, 64 * h, span.base, head, batch);
      }
    }
  };

  // Whether some row does not see some key of the tile from place n0 on (what
  // all rows see are one or two intervals of places).
  auto ragged = [&](int n0) {
    if (span.unplaced || n0 + KT > n_places) return true;
    const int a = min(span.sinks, span.hi0), l = s8 + span.lo1 - span.base, h = s8 + span.hi0 - span.base;
    return !(n0 + KT <= a || (n0 >= l && n0 + KT <= h) || (a >= l && n0 + KT <= h));
  };
  auto issue_k = [&](int j) {
    castdev::mbar_arrive_expect_tx(&k_full[j & 1], S::tile);
    start(smem + S::k_off + (j & 1) * S::tile, &k_full[j & 1], (kt_lo + j) * KT, &tm_k, &tm_k_sink, &tm_k_rest,
          hk * p.k_head, b * p.k_batch);
  };
  auto issue_v = [&](int j) {
    uint64_t *full = ragged((kt_lo + j) * KT) ? &v_raw[j & 1] : &v_full[j & 1];
    castdev::mbar_arrive_expect_tx(full, S::tile);
    start(smem + S::v_off + (j & 1) * S::tile, full, (kt_lo + j) * KT, &tm_v, &tm_v_sink, &tm_v_rest, hk * p.v_head,
          b * p.v_batch);
  };

  if (warp == kKWarp && lane == 0) {
    *err = 0;
    *bad_flag = 0;
    for (int i = 0; i < S::n_bars; ++i) castdev::mbar_init(&bar[i], 1);
    for (int i = 0; i < 2; ++i) castdev::mbar_init(&p_full[i], 4);
    castdev::fence_barrier_init();
    if (n_kv > 0) {  // what the first product needs, before the block meets
      castdev::mbar_arrive_expect_tx(q_full, S::q_tile);
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
        tma_load_5d(smem + h * 16384, &tm_q, q_full, 64 * h, 0, row0 >> p.pack_log2, hg, b);
      issue_k(0);
    }
  }
  if (warp == kMWarp) {
    castdev::tmem_alloc(tmem_slot, S::tmem_cols);
    castdev::tmem_relinquish();
  }
  __syncthreads();
  castdev::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp >= 4) {
    regs_dec<S::regs_rest>();
    if (warp == kKWarp) {
      if (lane == 0 && n_kv > 0) {
        int issued = 1;
        for (int j = 1; j < n_kv; ++j) {  // (the stage is free when S of step j - 2 is done)
          if (j >= 2 && !castdev::mbar_wait(&k_free[j & 1], ((j >> 1) - 1) & 1, err)) break;
          issue_k(j);
          issued = j + 1;
        }
        castdev::mbar_wait_drain(q_full, 0, err);
        for (int j = max(0, issued - 2); j < issued; ++j)
          castdev::mbar_wait_drain(&k_full[j & 1], (j >> 1) & 1, err);
      }
    } else if (warp == kVWarp) {
      // whole warp: lane 0 starts the copies, all go over tiles that are not wholly visible
      uint32_t raw_phase = 0;  // bit per stage
      // every row sees place n (sinks and the keys of all rows)
      auto all_see = [&](int n) {
        return !span.unplaced && (n < min(span.sinks, span.hi0) || (n >= s8 + span.lo1 - span.base && n < s8 + span.hi0 - span.base));
      };
      auto go_over = [&](int j) -> bool {
        const int n0 = (kt_lo + j) * KT, vs = j & 1;
        const bool ok = castdev::mbar_wait(&v_raw[vs], (raw_phase >> vs) & 1, err);
        if (!__all_sync(0xffffffffu, ok)) return false;
        raw_phase ^= 1u << vs;
        uint8_t *tile = smem + S::v_off + vs * S::tile;
        // rows that nobody sees: places [s_n, s8) and from n_places on
        auto zero = [&](int from, int to) {
          for (int r = max(from, 0) + (lane >> 3); r < min(to, KT); r += 4)
#pragma unroll
            for (int h = 0; h < D / 64; ++h)
              reinterpret_cast<uint4 *>(tile + h * S::half + r * 128)[lane & 7] = make_uint4(0u, 0u, 0u, 0u);
        };
        if (s8 > span.s_n) zero(span.s_n - n0, s8 - n0);
        zero(n_places - n0, KT);
        __syncwarp();
        // 0 * x is NaN for the values looked for, and only for them
        uint32_t acc = 0;
        const uint4 *w = reinterpret_cast<const uint4 *>(tile) + lane;
#pragma unroll
        for (int i0 = 0; i0 < S::tile / 512; i0 += 8) {
          uint4 u[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i] = w[(i0 + i) * 32];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            acc = Half2<T>::fma0(u[i].x, acc);
            acc = Half2<T>::fma0(u[i].y, acc);
            acc = Half2<T>::fma0(u[i].z, acc);
            acc = Half2<T>::fma0(u[i].w, acc);
          }
        }
        if (__any_sync(0xffffffffu, Half2<T>::bad(acc) != 0)) {
          bool bad = false;
          for (int r = lane >> 3; r < KT; r += 4) {  // eight lanes a row of 128 bytes
            if (all_see(n0 + r)) continue;
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
              uint4 *q = reinterpret_cast<uint4 *>(tile + h * S::half + r * 128) + (lane & 7);
              const uint4 u = *q;
              const uint32_t b0 = Half2<T>::bad(u.x), b1 = Half2<T>::bad(u.y), b2 = Half2<T>::bad(u.z),
                             b3 = Half2<T>::bad(u.w);
              if (b0 | b1 | b2 | b3) {
                bad = true;
                *q = make_uint4(u.x & ~b0, u.y & ~b1, u.z & ~b2, u.w & ~b3);
              }
            }
          }
          if (bad) *bad_flag = 1;
        }
        castdev::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) castdev::mbar_arrive(&v_full[vs]);
        return true;
      };
      int issued = min(n_kv, 2), looked = 0;  // tiles started; tiles gone over
      bool ok = true;
      if (lane == 0)
        for (int j = 0; j < issued; ++j) issue_v(j);
      for (int j = 0; ok && j < n_kv; ++j) {
        if (j >= 2) {  // (the stage is free when P V of step j - 2 is done)
          ok = __all_sync(0xffffffffu, castdev::mbar_wait(&v_free[j & 1], ((j >> 1) - 1) & 1, err));
          if (!ok) break;
          if (lane == 0) issue_v(j);
          issued = j + 1;
        }
        if (ragged((kt_lo + j) * KT)) ok = go_over(j);
        if (ok) looked = j + 1;
      }
      // every copy lands before the CTA leaves: those gone over have; the
      // others' own barriers say so
      if (lane == 0)
        for (int j = max(0, issued - 2); j < issued; ++j) {
          const int vs = j & 1;
          if (!ragged((kt_lo + j) * KT))
            castdev::mbar_wait_drain(&v_full[vs], (j >> 1) & 1, err);
          else if (j >= looked)
            castdev::mbar_wait_drain(&v_raw[vs], (raw_phase >> vs) & 1, err);
        }
    } else if (warp == kMWarp) {
      if (lane == 0 && n_kv > 0) {
        tiles_issuer<T, D>(tmem, castdev::smem_u32(smem), n_kv, q_full, k_full, v_full, s_full, p_full, pv_done, k_free, v_free, err);
        castdev::tc_commit(mma_drain);
        castdev::mbar_wait_drain(mma_drain, 0, err);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    regs_inc<S::regs_soft>();
    const int lrow = warp * 32 + lane;
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    const uint32_t o_addr = tmem + lane_off;
    const uint32_t s_addr = tmem + lane_off + S::s_col;
    const int my_steps = n_kv;
    const int row = row0 + lrow;
    const bool row_valid = row < p.rows;
    const int token = row >> p.pack_log2, head = hg * p.pack + (row & (p.pack - 1));
    // this row's places: [0, near) and [from, to)
    int lo = 0, hi = 0, near = 0, from = 0, to = 0;
    const int pos = len - p.Lq + token;
    if (row_valid && pos >= 0) {
      window_bounds(p.rule, len, pos, lo, hi);
      near = min(span.sinks, hi);
      from = s8 + lo - span.base;
      to = s8 + hi - span.base;
    }
    // what all rows of the warp see, and what none does (rows past the end are left out)
    const int big = 1 << 30;
    const int w_near_lo = __reduce_min_sync(0xffffffffu, row_valid ? near : big);
    const int w_near_hi = __reduce_max_sync(0xffffffffu, near);
    const int w_from_lo = __reduce_min_sync(0xffffffffu, row_valid ? from : big);
    const int w_from_hi = __reduce_max_sync(0xffffffffu, from);
    const int w_to_lo = __reduce_min_sync(0xffffffffu, row_valid ? to : big);
    const int w_to_hi = __reduce_max_sync(0xffffffffu, to);
    // (a row that will see nothing must not keep its warp on the slow path)
    float m_run = hi > 0 ? -INFINITY : 0.0f, l_run = 0.0f;
    bool ok = true;
    const float c2 = p.scale_log2;
    for (int h = 0; h < my_steps; ++h) {
      const int n0 = kt_lo * KT + h * 64;
      const bool full_step = n0 + 64 <= w_near_lo || (n0 >= w_from_hi && n0 + 64 <= w_to_lo);
      const bool empty_step = n0 >= w_near_hi && (n0 + 64 <= w_from_lo || n0 >= w_to_hi);
      uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
      if (!full_step) {
#pragma unroll
        for (int w = 0; w < 2; ++w)
          seen[w] = interval_mask(0, near, n0 + 32 * w) | interval_mask(from, to, n0 + 32 * w);
      }
      ok = __all_sync(0xffffffffu, castdev::mbar_wait(&s_full[S::buf(h)], S::phase(h), err));
      if (!ok) break;
      castdev::tc_fence_after();
      const uint32_t sb = s_addr + 64 * S::buf(h);
      float sum = 0.0f;
      // Raises the running maximum to a row's mx where that is above it by more
      // than the slack, and scales what is relative to it: l, O and the sum of
      // this step.  The maximum is a whole number, so all of that, P included,
      // is scaled by powers of two.  Returns the scale (1: not raised).
      auto raise = [&](float mx) -> float {
        float f = 1.0f;
        if (mx > m_run + X::kSlack || m_run == -INFINITY) {
          const float m_new = fmaxf(m_run, ceilf(mx));
          f = (m_run == -INFINITY) ? (m_new == -INFINITY ? 1.0f : 0.0f) : fast_exp2(m_run - m_new);
          l_run *= f;
          sum *= f;
          m_run = m_new;
        }
        if (h > 0 && __any_sync(0xffffffffu, f != 1.0f)) {
          ok = __all_sync(0xffffffffu, castdev::mbar_wait(&pv_done[S::buf(h - 1)], S::phase(h - 1), err));
          if (ok) {
            castdev::tc_fence_after();
#pragma unroll 1
            for (int cc = 0; cc < D / 32; ++cc) {
              uint32_t o[32];
              tmem_get(o_addr + 32 * cc, o);
#pragma unroll
              for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
              tmem_put(o_addr + 32 * cc, o);
            }
            // (the second chunk of a step may raise the maximum again and read O)
            castdev::tmem_wait_st();
          }
        }
        return f;
      };
      auto find = [&](uint32_t addr, int words, const uint32_t *w) -> float {  // maximum of 32 * words scores in TMEM
        float mx = -INFINITY;
#pragma unroll 1
        for (int q = 0; q < words; ++q) {
          uint32_t x[32];
          tmem_get(addr + 32 * q, x);
          mx = fmaxf(mx, tiles_max(x, q ? w[1] : w[0], c2));
        }
        return mx;
      };
      if (empty_step) {
        const uint32_t zero[16] = {};
        tmem_put(sb, zero);
        tmem_put(sb + 16, zero);
      } else {
        if (__builtin_expect(__any_sync(0xffffffffu, m_run == -INFINITY), 0)) raise(find(sb, 2, seen));
        // A chunk of columns at a time.  P of the first chunk goes over scores
        // that have been read.
#pragma unroll 1
        for (int q = 0; q < 64 / S::chunk; ++q) {
          uint32_t x[S::chunk], pk[S::chunk / 2], mine[S::chunk / 32];
          if constexpr (S::chunk == 64) {
            mine[0] = seen[0], mine[1] = seen[1];
          } else {
            mine[0] = q ? seen[1] : seen[0];
          }
          float part;
          for (bool again = false;;) {
            tmem_get(sb + S::chunk * q, x);
            const float base = (m_run == -INFINITY) ? 0.0f : m_run - X::kShift;
            part = full_step ? tiles_probs<T, false, S::chunk>(x, pk, mine, c2, base)
                             : tiles_probs<T, true, S::chunk>(x, pk, mine, c2, base);
            if (again || !__any_sync(0xffffffffu, !(part <= X::kSumLimit))) break;
            // some weights are too large against a maximum that is behind: it
            // is found, and the pass made again
            const float f = raise(find(sb + S::chunk * q, S::chunk / 32, mine));
            if (S::chunk == 32 && q == 1) {  // the first chunk's P, already stored
              uint32_t w[16];
              castdev::tmem_wait_st();
              tmem_get(sb, w);
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                const float2 y = Half2<T>::unpack(w[c]);
                w[c] = X::pack(y.x * f, y.y * f);
              }
              tmem_put(sb, w);
            }
            again = true;
          }
          tmem_put(sb + S::chunk / 2 * q, pk);
          sum += part;
        }
        if (!ok) break;
      }
      l_run += sum;
      castdev::tmem_wait_st();
      castdev::tc_fence_before();
      __syncwarp();
      if (lane == 0) castdev::mbar_arrive(&p_full[S::buf(h)]);
    }
    if (hi == 0) {  // a row that sees nothing is nothing (and its maximum is none)
      m_run = -INFINITY;
      l_run = 0.0f;
    }
    // ------------------------------------------------------------ epilogue
    if (ok && my_steps > 0) {
      const int hl = my_steps - 1;
      ok = __all_sync(0xffffffffu, castdev::mbar_wait(&pv_done[S::buf(hl)], S::phase(hl), err));
      castdev::tc_fence_after();
    }
    {
      auto load_o = [&](int cc, uint32_t (&o)[32]) {
        if (my_steps > 0) {
          castdev::tmem_ld32(o_addr + 32 * cc, o);
          castdev::tmem_wait_ld();
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = 0u;
        }
      };
      const bool bad = *bad_flag != 0;
      if (n_parts == 1) {
        if (ok) {
          const float inv = l_run != 0.0f ? 1.0f / l_run : 0.0f;  // (a NaN sum stays one)
          // Rows go to the Q tile's place in shared memory, swizzled as the
          // map wants them (no product reads Q any more), and out by one copy,
          // which leaves out rows past the last token.
#pragma unroll 1
          for (int cc = 0; cc < D / 32; ++cc) {
            uint32_t o[32];
            __syncwarp();
            load_o(cc, o);
            float y[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) y[c] = hi > 0 ? __uint_as_float(o[c]) * inv : 0.0f;
            if (__builtin_expect(bad, 0) && row_valid) {
              float z[32];
              for (int c = 0; c < 32; ++c) z[c] = y[c];
              tiles_give_back<T>(p, span, b, hk, lo, hi, 32 * cc, z);
              for (int c = 0; c < 32; ++c) y[c] = z[c];
            }
            uint8_t *line = smem + (cc >> 1) * 16384 + lrow * 128;
#pragma unroll
            for (int c = 0; c < 4; ++c)
              *reinterpret_cast<uint4 *>(line + (((4 * (cc & 1) + c) ^ (lrow & 7)) * 16)) =
                  make_uint4(X::pack(y[8 * c], y[8 * c + 1]), X::pack(y[8 * c + 2], y[8 * c + 3]),
                             X::pack(y[8 * c + 4], y[8 * c + 5]), X::pack(y[8 * c + 6], y[8 * c + 7]));
          }
        }
        castdev::fence_proxy_async_smem();
        castdev::named_bar_sync(1, 128);
        if (threadIdx.x == 0 && ok) {
#pragma unroll
          for (int h = 0; h < D / 64; ++h) tma_store_5d(&tm_o, smem + h * 16384, 64 * h, 0, row0 >> p.pack_log2, hg, b);
          asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        }
      } else if (ok) {
        // this part's O, maximum and sum: [tile][column][row], then [tile][m, l, flag][row]
        float *slot = p.part + (long long)(blockIdx.x - p.n_whole) * tiles_part_floats<D>();
        float *tail = slot + 128 * D + lrow;
        if (row_valid) {
          tail[0] = hi > 0 ? m_run : -INFINITY;
          tail[128] = l_run;
          tail[256] = __int_as_float(bad ? 1 : 0);
        }
        if (my_steps > 0) {
#pragma unroll 1
          for (int cc = 0; cc < D / 32; ++cc) {
            uint32_t o[32];
            __syncwarp();
            load_o(cc, o);
            float *dst = slot + 32 * cc * 128 + lrow;
            if (row_valid) {
#pragma unroll
              for (int c = 0; c < 32; ++c) dst[c * 128] = __uint_as_float(o[c]);
            }
          }
        }
      }
    }
  }
  __syncthreads();
  if (warp == kMWarp) {
    castdev::tc_fence_after();
    castdev::tmem_dealloc(tmem, S::tmem_cols);
  }
}

// Joins the parts of the cut items: one CTA for eight columns of a query tile;
// thread (row, g) takes every kJoinGroups-th part, several loads at a time.
constexpr int kJoinCols = 8;
template <typename T, int D, int kJoinGroups>
__global__ void __launch_bounds__(128 * kJoinGroups) window_tiles_join_kernel(const __grid_constant__ TilesParams p) {
  __shared__ float acc_s[kJoinGroups][kJoinCols + 1][128];
  __shared__ float max_s[kJoinGroups][128];
  constexpr int cuts = D / kJoinCols;
  constexpr long long kPart = tiles_part_floats<D>();
  const int cut = blockIdx.x % cuts, item = blockIdx.x / cuts;
  const int row_in = threadIdx.x & 127, g = threadIdx.x >> 7;
  const int x = p.n_whole + item;
  const int bhg = p.by_tiles.div(x), qt = p.q_tiles - 1 - (x - bhg * p.q_tiles);
  const int b = p.by_groups.div(bhg), hg = bhg - b * p.head_groups;
  const int row0 = qt * 128, row_end = min(p.rows, row0 + 128);
  const int row = row0 + row_in;
  const bool on = row < p.rows;
  const float *base = p.part + (long long)item * p.parts * kPart;
  const float *tails = base + 128 * D + row_in;
  const int parts = on ? p.parts : 0;
  float m = -INFINITY, l = 0.0f, a[kJoinCols];
#pragma unroll
  for (int c = 0; c < kJoinCols; ++c) a[c] = 0.0f;
  bool bad = false;
  constexpr int kAtOnce = 3;  // parts whose loads are under way together
  for (int j0 = g; j0 < parts; j0 += kAtOnce * kJoinGroups) {
    float mj[kAtOnce], lj[kAtOnce], flag[kAtOnce], v[kAtOnce][kJoinCols];
    float top = m;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int j = min(j0 + u * kJoinGroups, parts - 1);
      const float *tail = tails + j * kPart, *o = base + j * kPart + cut * kJoinCols * 128 + row_in;
      mj[u] = j0 + u * kJoinGroups < parts ? __ldg(tail) : -INFINITY;
      lj[u] = __ldg(tail + 128), flag[u] = __ldg(tail + 256);
#pragma unroll
      for (int c = 0; c < kJoinCols; ++c) v[u][c] = __ldg(o + c * 128);
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      top = fmaxf(top, mj[u]);
      bad = bad || __float_as_int(flag[u]) != 0;
    }
    const float f0 = m == -INFINITY ? 0.0f : fast_exp2(m - top);
    m = top;
    l *= f0;
#pragma unroll
    for (int c = 0; c < kJoinCols; ++c) a[c] *= f0;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      // Nothing was seen (O may hold anything), or nothing but NaN scores: these
      // leave no maximum and a NaN sum, which makes the row NaN.
      if (mj[u] == -INFINITY) {
        if (isnan(lj[u])) l = lj[u];
        continue;
      }
      const float f = fast_exp2(mj[u] - m);
      l = fmaf(lj[u], f, l);
#pragma unroll
      for (int c = 0; c < kJoinCols; ++c) a[c] = fmaf(v[u][c], f, a[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < kJoinCols; ++c) acc_s[g][c][row_in] = a[c];
  acc_s[g][kJoinCols][row_in] = l;
  max_s[g][row_in] = m;
  const bool any_bad = __syncthreads_or(bad);
  if (g != 0 || !on) return;
  float y[kJoinCols];
  l = 0.0f;
#pragma unroll
  for (int c = 0; c < kJoinCols; ++c) y[c] = 0.0f;
#pragma unroll
  for (int j = 0; j < kJoinGroups; ++j) m = fmaxf(m, max_s[j][row_in]);
#pragma unroll
  for (int j = 0; j < kJoinGroups; ++j) {
    const float mj = max_s[j][row_in], f = mj == -INFINITY ? 0.0f : fast_exp2(mj - m);
    l = fmaf(acc_s[j][kJoinCols][row_in], f, l);
#pragma unroll
    for (int c = 0; c < kJoinCols; ++c) y[c] = fmaf(acc_s[j][c][row_in], f, y[c]);
  }
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
  for (int c = 0; c < kJoinCols; ++c) y[c] *= inv;
  const int token = row >> p.pack_log2, head = hg * p.pack + (row & (p.pack - 1));
  if (any_bad) {
    const int len = min(max(p.kv_lens ? p.kv_lens[b] : p.lk, 0), p.lk);
    const WindowSpan span = window_span(p.rule, len, p.Lq, row0 >> p.pack_log2, (row_end - 1) >> p.pack_log2);
    int lo = 0, hi = 0;
    const int pos = len - p.Lq + token;
    if (pos >= 0) window_bounds(p.rule, len, pos, lo, hi);
    float z[kJoinCols];
    for (int c = 0; c < kJoinCols; ++c) z[c] = y[c];
    tiles_give_back<T>(p, span, b, p.by_keys.div(hg), lo, hi, cut * kJoinCols, z);
    for (int c = 0; c < kJoinCols; ++c) y[c] = z[c];
  }
  T *dst = static_cast<T *>(p.out) + b * p.os[0] + head * p.os[1] + token * p.os[2] + cut * kJoinCols;
  *reinterpret_cast<uint4 *>(dst) =
      make_uint4(TilesType<T>::pack(y[0], y[1]), TilesType<T>::pack(y[2], y[3]), TilesType<T>::pack(y[4], y[5]),
                 TilesType<T>::pack(y[6], y[7]));
}

}  // namespace castk
