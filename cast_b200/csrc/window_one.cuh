// Window attention, one 128-row query tile a CTA, two CTAs an SM.
#pragma once

#include "window_tiles.cuh"

namespace castk {

constexpr int kOneThreads = 256;
constexpr int kOneRegsSoft = 200, kOneRegsRest = 56;  // 128 (200 + 56) = 256 * 128, the launch's registers

template <int D>
struct OneSmem {
  static constexpr int keys = D == 128 ? 64 : 128;  // of one K or V tile
  static constexpr int q_tile = 128 * D * 2;
  static constexpr int tile = keys * D * 2;         // 16 KB
  static constexpr int half = keys * 128;           // 64 columns of a tile
  static constexpr int kStages = 2, vStages = 3;
  static constexpr int k_off = q_tile;
  static constexpr int v_off = k_off + kStages * tile;
  static constexpr int bars = v_off + vStages * tile;
  // q_full, k_full/empty, v_full/empty/raw, s_full[2], p_full[2], pv_done[2], drain
  static constexpr int n_bars = 1 + 2 * kStages + 3 * vStages + 6 + 1;
  static constexpr int tmem_slot = bars + 8 * n_bars;
  static constexpr int alloc = tmem_slot + 16;
};

template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Issues the products of one query tile over n 64-key steps.  S of step h + 2
// goes into the buffer that P of step h came from, right after P V of step h.
template <typename T, int D>
__device__ __forceinline__ bool one_issuer(uint32_t tmem, uint32_t sbase, int n, uint64_t *q_full, uint64_t *k_full,
                                           uint64_t *k_empty, uint64_t *v_full, uint64_t *v_empty, uint64_t *s_full,
                                           uint64_t *p_full, uint64_t *pv_done, int *err) {
  using S = OneSmem<D>;
  constexpr int KS = S::kStages, VS = S::vStages, HT = S::keys / 64;
  constexpr uint32_t fmt = TilesType<T>::fmt;
  constexpr uint32_t idesc_s = castdev::make_idesc(1, fmt, fmt, 0, 0, 128, 64);
  constexpr uint32_t idesc_pv = castdev::make_idesc(1, fmt, fmt, 0, 1, 128, D);
  const DescW qd = desc_words(sbase, 16);
  const DescW kd = desc_words(sbase + S::k_off, 16);
  const DescW vd = desc_words(sbase + S::v_off, S::half);
  const uint32_t s_col = tmem + 128;
  auto issue_s = [&](int h) {  // false: a wait gave up
    const int t = h / HT, sub = h % HT, ks = t % KS;
    if (sub == 0) {
      if (!castdev::mbar_wait(&k_full[ks], (t / KS) & 1, err)) return false;
      castdev::tc_fence_after();
    }
    const uint32_t d = s_col + (h & 1) * 64, ko = ks * S::tile + sub * 8192;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
      castdev::mma_f16_ss(d, qd.at((s >> 2) * 16384 + (s & 3) * 32), kd.at(ko + (s >> 2) * S::half + (s & 3) * 32),
                          idesc_s, s > 0);
    castdev::tc_commit(&s_full[h & 1]);
    if (sub == HT - 1) castdev::tc_commit(&k_empty[ks]);
    return true;
  };
  if (!castdev::mbar_wait(q_full, 0, err)) return false;
  if (!issue_s(0) || (n > 1 && !issue_s(1))) return false;
  for (int h = 0; h < n; ++h) {
    const int t = h / HT, sub = h % HT, vs = t % VS;
    if (sub == 0 && !castdev::mbar_wait(&v_full[vs], (t / VS) & 1, err)) return false;
    if (!castdev::mbar_wait(&p_full[h & 1], (h >> 1) & 1, err)) return false;
    castdev::tc_fence_after();
    const uint32_t vo = vs * S::tile + sub * 8192, pa = s_col + (h & 1) * 64;
#pragma unroll
    for (int s = 0; s < 4; ++s) castdev::mma_f16_ts(tmem, pa + 8 * s, vd.at(vo + 2048 * s), idesc_pv, (h | s) != 0);
    castdev::tc_commit(&pv_done[h & 1]);
    if (sub == HT - 1) castdev::tc_commit(&v_empty[vs]);
    if (h + 2 < n && !issue_s(h + 2)) return false;
  }
  return true;
}

template <int D>
__host__ __device__ constexpr long long one_part_floats() {
  return 128ll * (D + kTilesPartCols);
}

template <typename T, int D>
__global__ void __launch_bounds__(kOneThreads, 2)
    window_one_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                        const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_k_sink,
                        const __grid_constant__ CUtensorMap tm_v_sink, const __grid_constant__ CUtensorMap tm_k_rest,
                        const __grid_constant__ CUtensorMap tm_v_rest, const __grid_constant__ TilesParams p) {
  using S = OneSmem<D>;
  using X = TilesType<T>;
  constexpr int KS = S::kStages, VS = S::vStages;
  constexpr int KT = S::keys;
  extern __shared__ __align__(1024) uint8_t smem_one[];
  uint8_t *smem = smem_one;
  uint64_t *bar = reinterpret_cast<uint64_t *>(smem + S::bars);
  uint64_t *q_full = bar;
  uint64_t *k_full = bar + 1;
  uint64_t *k_empty = k_full + KS;
  uint64_t *v_full = k_empty + KS;
  uint64_t *v_empty = v_full + VS;
  uint64_t *v_raw = v_empty + VS;  // a V tile has landed and is gone over before v_full
  uint64_t *s_full = v_raw + VS;
  uint64_t *p_full = s_full + 2;
  uint64_t *pv_done = p_full + 2;
  uint64_t *mma_drain = pv_done + 2;
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
  const int bhg = x / p.q_tiles;
  const int qt = p.q_tiles - 1 - (x - bhg * p.q_tiles);  // later rows see more keys: first
  const int b = bhg / p.head_groups, hg = bhg - b * p.head_groups;
  const int hk = hg / p.groups_per_key;
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
  const int kt_lo = (int)((long long)part * n_tiles / n_parts);
  const int n_kv = (int)((long long)(part + 1) * n_tiles / n_parts) - kt_lo;
  constexpr int kKWarp = 4, kMWarp = 5, kVWarp = 6;

  if (warp == kKWarp && lane == 0) {
    *err = 0;
    *bad_flag = 0;
    for (int i = 0; i < S::n_bars; ++i) castdev::mbar_init(&bar[i], 1);
    for (int i = 0; i < 2; ++i) castdev::mbar_init(&p_full[i], 4);
    castdev::fence_barrier_init();
    castdev::tma_prefetch_desc(&tm_q);
    castdev::tma_prefetch_desc(&tm_k);
    castdev::tma_prefetch_desc(&tm_v);
    if (n_kv > 0) {
      castdev::mbar_arrive_expect_tx(q_full, S::q_tile);
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
        tma_load_5d(smem + h * 16384, &tm_q, q_full, 64 * h, 0, row0 >> p.pack_log2, hg, b);
    }
  }
  if (warp == kMWarp) {
    castdev::tmem_alloc(tmem_slot, 256);
    castdev::tmem_relinquish();
  }
  __syncthreads();
  castdev::tc_fence_after();
  const uint32_t tmem = *tmem_slot;

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

  if (warp >= 4) {
    regs_dec<kOneRegsRest>();
    if (warp == kKWarp) {
      if (lane == 0 && n_kv > 0) {
        int issued = 0;
        for (int j = 0; j < n_kv; ++j) {
          const int n0 = (kt_lo + j) * KT, ks = j % KS;
          if (j >= KS && !castdev::mbar_wait(&k_empty[ks], ((j / KS) - 1) & 1, err)) break;
          castdev::mbar_arrive_expect_tx(&k_full[ks], S::tile);
          start(smem + S::k_off + ks * S::tile, &k_full[ks], n0, &tm_k, &tm_k_sink, &tm_k_rest, hk * p.k_head,
                b * p.k_batch);
          issued = j + 1;
        }
        castdev::mbar_wait_drain(q_full, 0, err);
        for (int j = max(0, issued - KS); j < issued; ++j)
          castdev::mbar_wait_drain(&k_full[j % KS], (j / KS) & 1, err);
      }
    } else if (warp == kVWarp) {
      // whole warp: lane 0 starts the copies, all go over tiles that are not wholly visible
      uint32_t raw_phase = 0;  // bit per stage
      // every row sees place n (sinks and the keys of all rows)
      auto all_see = [&](int n) {
        return !span.unplaced && (n < min(span.sinks, span.hi0) || (n >= s8 + span.lo1 - span.base && n < s8 + span.hi0 - span.base));
      };
      // (both ends of a run of KT places: visible ones are one or two intervals)
      auto ragged = [&](int n0) {
        if (span.unplaced || n0 + KT > n_places) return true;
        const int a = min(span.sinks, span.hi0), l = s8 + span.lo1 - span.base, h = s8 + span.hi0 - span.base;
        return !(n0 + KT <= a || (n0 >= l && n0 + KT <= h) || (a >= l && n0 + KT <= h));
      };
      auto go_over = [&](int j) -> bool {
        const int n0 = (kt_lo + j) * KT, vs = j % VS;
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
      int issued = 0, looked = 0;  // tiles started; tiles gone over
      bool ok = true;
      for (int j = 0; ok && j < n_kv; ++j) {
        const int n0 = (kt_lo + j) * KT, vs = j % VS;
        ok = j < VS || castdev::mbar_wait(&v_empty[vs], ((j / VS) - 1) & 1, err);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        uint64_t *full = ragged(n0) ? &v_raw[vs] : &v_full[vs];
        if (lane == 0) {
          castdev::mbar_arrive_expect_tx(full, S::tile);
          start(smem + S::v_off + vs * S::tile, full, n0, &tm_v, &tm_v_sink, &tm_v_rest, hk * p.v_head, b * p.v_batch);
        }
        issued = j + 1;
        if (j > 0) {
          if (ragged((kt_lo + j - 1) * KT)) ok = go_over(j - 1);
          looked = j;
        }
      }
      if (ok && issued > 0 && ragged((kt_lo + issued - 1) * KT)) ok = go_over(issued - 1);
      if (ok) looked = issued;
      // every copy lands before the CTA leaves: those gone over have; the
      // others' own barriers say so
      if (lane == 0)
        for (int j = max(0, issued - VS); j < issued; ++j) {
          const int vs = j % VS;
          if (!ragged((kt_lo + j) * KT))
            castdev::mbar_wait_drain(&v_full[vs], (j / VS) & 1, err);
          else if (j >= looked)
            castdev::mbar_wait_drain(&v_raw[vs], (raw_phase >> vs) & 1, err);
        }
    } else if (warp == kMWarp) {
      if (lane == 0 && n_kv > 0) {
        one_issuer<T, D>(tmem, castdev::smem_u32(smem), n_kv * (KT / 64), q_full, k_full, k_empty, v_full, v_empty,
                         s_full, p_full, pv_done, err);
        castdev::tc_commit(mma_drain);
        castdev::mbar_wait_drain(mma_drain, 0, err);
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    regs_inc<kOneRegsSoft>();
    const int lrow = warp * 32 + lane;
    const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
    const uint32_t o_addr = tmem + lane_off;
    const uint32_t s_addr = tmem + lane_off + 128;
    const int my_steps = n_kv * (KT / 64);
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
    // (a row that will see nothing must not keep its warp on the slow path)
    float m_run = hi > 0 ? -INFINITY : 0.0f, l_run = 0.0f;
    bool ok = true;
    const float c2 = p.scale_log2;
    for (int h = 0; h < my_steps; ++h) {
      const int half = h & 1;
      const int n0 = kt_lo * KT + h * 64;
      const bool all = n0 + 64 <= near || (n0 >= from && n0 + 64 <= to) || !row_valid;
      const bool none = (n0 >= near && (n0 + 64 <= from || n0 >= to)) || !row_valid;
      const bool full_step = __all_sync(0xffffffffu, all);
      const bool empty_step = __all_sync(0xffffffffu, none);
      uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
      if (!full_step) {
#pragma unroll
        for (int w = 0; w < 2; ++w)
          seen[w] = interval_mask(0, near, n0 + 32 * w) | interval_mask(from, to, n0 + 32 * w);
      }
      ok = __all_sync(0xffffffffu, castdev::mbar_wait(&s_full[half], (h >> 1) & 1, err));
      if (!ok) break;
      castdev::tc_fence_after();
      const uint32_t sb = s_addr + 64 * half;
      uint32_t v[64];
      float sum = 0.0f;
      if (empty_step) {
#pragma unroll
        for (int c = 0; c < 32; ++c) v[c] = 0u;
      } else {
        castdev::tmem_ld32(sb, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
        castdev::tmem_ld32(sb + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
        castdev::tmem_wait_ld();
        bool slow = __any_sync(0xffffffffu, m_run == -INFINITY);
        if (!slow) {
          sum = full_step ? tiles_probs<T, false>(v, seen, c2, m_run - X::kShift)
                          : tiles_probs<T, true>(v, seen, c2, m_run - X::kShift);
          slow = __any_sync(0xffffffffu, !(sum <= X::kSumLimit));
          if (slow) {
            castdev::tmem_ld32(sb, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
            castdev::tmem_ld32(sb + 32, *reinterpret_cast<uint32_t(*)[32]>(&v[32]));
            castdev::tmem_wait_ld();
          }
        }
        if (__builtin_expect(slow, 0)) {
          const float m_step = full_step ? row_max<false, false>(v, seen, c2) : row_max<false, true>(v, seen, c2);
          float o_scale = 1.0f;
          if (m_step > m_run + X::kSlack || m_run == -INFINITY) {
            const float m_new = fmaxf(m_run, m_step);
            o_scale = (m_run == -INFINITY) ? (m_new == -INFINITY ? 1.0f : 0.0f) : fast_exp2(m_run - m_new);
            l_run *= o_scale;
            m_run = m_new;
          }
          if (h > 0 && __any_sync(0xffffffffu, o_scale != 1.0f)) {
            const int hp = h - 1;
            ok = __all_sync(0xffffffffu, castdev::mbar_wait(&pv_done[hp & 1], (hp >> 1) & 1, err));
            if (!ok) break;
            castdev::tc_fence_after();
#pragma unroll 1
            for (int cc = 0; cc < D / 32; ++cc) {
              uint32_t o[32];
              castdev::tmem_ld32(o_addr + 32 * cc, o);
              castdev::tmem_wait_ld();
#pragma unroll
              for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * o_scale);
              castdev::tmem_st32(o_addr + 32 * cc, o);
            }
          }
          const float base = (m_run == -INFINITY) ? 0.0f : m_run - X::kShift;
          sum = full_step ? tiles_probs<T, false>(v, seen, c2, base) : tiles_probs<T, true>(v, seen, c2, base);
        }
      }
      castdev::tmem_st32(sb, *reinterpret_cast<uint32_t(*)[32]>(&v[0]));
      l_run += sum;
      castdev::tmem_wait_st();
      castdev::tc_fence_before();
      __syncwarp();
      if (lane == 0) castdev::mbar_arrive(&p_full[half]);
    }
    if (hi == 0) {  // a row that sees nothing is nothing (and its maximum is none)
      m_run = -INFINITY;
      l_run = 0.0f;
    }
    // ------------------------------------------------------------ epilogue
    if (ok && my_steps > 0) {
      const int hl = my_steps - 1;
      ok = __all_sync(0xffffffffu, castdev::mbar_wait(&pv_done[hl & 1], (hl >> 1) & 1, err));
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
          T *dst = static_cast<T *>(p.out) + b * p.os[0] + head * p.os[1] + token * p.os[2];
#pragma unroll 1
          for (int cc = 0; cc < D / 32; ++cc) {
            uint32_t o[32];
            __syncwarp();
            load_o(cc, o);
            float y[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) y[c] = hi > 0 ? __uint_as_float(o[c]) * inv : 0.0f;
            if (row_valid) {
              if (__builtin_expect(bad, 0)) {
                float z[32];
                for (int c = 0; c < 32; ++c) z[c] = y[c];
                tiles_give_back<T>(p, span, b, hk, lo, hi, 32 * cc, z);
                for (int c = 0; c < 32; ++c) y[c] = z[c];
              }
              uint4 w[4];
              uint32_t *wp = reinterpret_cast<uint32_t *>(w);
#pragma unroll
              for (int c = 0; c < 16; ++c) wp[c] = X::pack(y[2 * c], y[2 * c + 1]);
#pragma unroll
              for (int c = 0; c < 4; ++c) reinterpret_cast<uint4 *>(dst + 32 * cc)[c] = w[c];
            }
          }
        }
      } else if (ok) {
        // this part's O, maximum and sum: [tile][column][row], then [tile][m, l, flag][row]
        float *slot = p.part + (long long)(blockIdx.x - p.n_whole) * one_part_floats<D>();
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
    castdev::tmem_dealloc(tmem, 256);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(128 * kJoinGroups) window_one_join_kernel(const __grid_constant__ TilesParams p) {
  __shared__ float acc_s[kJoinGroups][kJoinCols + 1][128];
  constexpr int cuts = D / kJoinCols;
  const int cut = blockIdx.x % cuts, item = blockIdx.x / cuts;
  const int row_in = threadIdx.x & 127, g = threadIdx.x >> 7;
  const int x = p.n_whole + item;
  const int bhg = x / p.q_tiles, qt = p.q_tiles - 1 - (x - bhg * p.q_tiles);
  const int b = bhg / p.head_groups, hg = bhg - b * p.head_groups;
  const int row0 = qt * 128, row_end = min(p.rows, row0 + 128);
  const int row = row0 + row_in;
  const bool on = row < p.rows;
  const float *base = p.part + (long long)item * p.parts * one_part_floats<D>();
  const float *tails = base + 128 * D + row_in;
  float m = -INFINITY;
  bool bad = false;
  if (on)
    for (int j = 0; j < p.parts; ++j) m = fmaxf(m, tails[j * one_part_floats<D>()]);
  float l = 0.0f, a[kJoinCols];
#pragma unroll
  for (int c = 0; c < kJoinCols; ++c) a[c] = 0.0f;
  if (on) {
#pragma unroll 4
    for (int j = g; j < p.parts; j += kJoinGroups) {
      const float *tail = tails + j * one_part_floats<D>();
      const float mj = tail[0];
      bad = bad || __float_as_int(tail[256]) != 0;
      if (mj == -INFINITY) continue;  // nothing seen: its O may not be written
      const float f = fast_exp2(mj - m);
      const float *o = base + j * one_part_floats<D>() + cut * kJoinCols * 128 + row_in;
      l = fmaf(tail[128], f, l);
#pragma unroll
      for (int c = 0; c < kJoinCols; ++c) a[c] = fmaf(o[c * 128], f, a[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < kJoinCols; ++c) acc_s[g][c][row_in] = a[c];
  acc_s[g][kJoinCols][row_in] = l;
  const bool any_bad = __syncthreads_or(bad);
  if (g != 0 || !on) return;
  float y[kJoinCols];
  l = 0.0f;
#pragma unroll
  for (int c = 0; c < kJoinCols; ++c) y[c] = 0.0f;
#pragma unroll
  for (int j = 0; j < kJoinGroups; ++j) {
    l += acc_s[j][kJoinCols][row_in];
#pragma unroll
    for (int c = 0; c < kJoinCols; ++c) y[c] += acc_s[j][c][row_in];
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
    tiles_give_back<T>(p, span, b, hg / p.groups_per_key, lo, hi, cut * kJoinCols, z);
    for (int c = 0; c < kJoinCols; ++c) y[c] = z[c];
  }
  T *dst = static_cast<T *>(p.out) + b * p.os[0] + head * p.os[1] + token * p.os[2] + cut * kJoinCols;
  *reinterpret_cast<uint4 *>(dst) =
      make_uint4(TilesType<T>::pack(y[0], y[1]), TilesType<T>::pack(y[2], y[3]), TilesType<T>::pack(y[4], y[5]),
                 TilesType<T>::pack(y[6], y[7]));
}

}  // namespace castk
