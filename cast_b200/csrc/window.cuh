// Sliding-window attention with visible first tokens (sinks), for few query
// rows: a split over the keys, dense or paged.
//
// Query i of Lq (position p = len - Lq + i of a session of len keys) sees key
// j < len with f(j) <= f(p) and (f(j) > f(p) - window or f(j) < sinks), where
// f(x) = x / frame: the keys [lo(p), hi(p)) and the sinks [0, S),
//   hi(p) = min(len, (f(p) + 1) frame), lo(p) = max(0, (f(p) - window + 1) frame),
//   S = sinks * frame.
// Both bounds grow with p, so the rows of a tile together see one list of
// keys: the S sinks followed by [lo(first row), hi(last row)), or [0, hi)
// where the two meet.  A place in that list is a "virtual" key.
//
// out = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m), s_j = q.k_j scale log2(e),
// in one pass over the keys with a running m.
#pragma once

#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "attention.cuh"
#include "common.cuh"

namespace castk {

// ------------------------------------------------------------------ masks
// n / d for 0 <= n < 2^31 by a product: with l = ceil(log2 d),
// floor(2^(31 + l) / d) + 1 exceeds 2^(31 + l) / d by at most 1, which moves
// the quotient of n < 2^31 by less than 1 / d (d = 1: n itself).
struct FastDiv {
  uint32_t d, mul, shift;
  void set(uint32_t v) {
    d = v;
    uint32_t l = 0;
    while ((1ull << l) < v) ++l;
    mul = v == 1 ? 0u : (uint32_t)((1ull << (31 + l)) / v + 1);
    shift = l - 1;
  }
  __device__ __forceinline__ int div(int n) const {
    return d == 1 ? n : (int)(__umulhi((uint32_t)n, mul) >> shift);
  }
};

// Frames, and keys of the sinks; lengths and positions are below 2^30, and so
// are the numbers here (what is larger means the same as 2^30), so that no
// bound of a window passes 31 bits.
struct WindowRule {
  int window, frame, sink_keys;
  FastDiv by_frame;
  void set(long long window_frames, long long sink_frames, int frame_tokens) {
    const long long most = 1ll << 30;
    window = (int)std::min(window_frames, most);
    frame = (int)std::min<long long>(frame_tokens, most);
    sink_keys = (int)std::min(std::min(sink_frames, most) * frame, most);
    by_frame.set((uint32_t)frame);
  }
};

// What the rows of one tile see of a session of `len` keys.
struct WindowSpan {
  int len, lq;
  int sinks;      // S, clipped to len
  int s_n;        // virtual keys that are sinks (0 where the list is contiguous)
  int base;       // key of virtual key s_n
  int n;          // virtual keys
  int lo0, hi0;   // lo, hi of the first row that has a position
  int lo1, hi1;   // of the last row
  bool unplaced;  // some row has no position (it sees nothing)
  __device__ __forceinline__ int key(int v) const { return v < s_n ? v : base + (v - s_n); }
  // whether a key of the list is hidden from some row of the tile
  __device__ __forceinline__ bool some(int key) const {
    return unplaced || key >= hi0 || (key >= sinks && key < lo1);
  }
};

__device__ __forceinline__ void window_bounds(const WindowRule &r, int len, int p, int &lo, int &hi) {
  const int f = r.by_frame.div(p);
  hi = min((f + 1) * r.frame, len);
  const int l = f + 1 - r.window;  // first visible frame
  lo = l <= 0 ? 0 : min(l * r.frame, len);
}

// Rows i0 .. i1 (inclusive) of lq queries.
__device__ __forceinline__ WindowSpan window_span(const WindowRule &r, int len, int lq, int i0, int i1) {
  WindowSpan s;
  s.len = len;
  s.lq = lq;
  s.sinks = min(r.sink_keys, len);
  s.s_n = s.base = s.n = s.lo0 = s.hi0 = s.lo1 = s.hi1 = 0;
  s.unplaced = len - lq + i0 < 0;
  const int p1 = len - lq + i1;
  if (p1 < 0) return s;  // no row of the tile has a position
  const int p0 = max(0, len - lq + i0);
  window_bounds(r, len, p0, s.lo0, s.hi0);
  window_bounds(r, len, p1, s.lo1, s.hi1);
  if (s.sinks < s.lo0) {
    s.s_n = s.sinks;
    s.base = s.lo0;
  }
  s.n = s.s_n + s.hi1 - s.base;
  return s;
}

__device__ __forceinline__ bool window_sees(int key, int lo, int hi, int sinks) {
  return key < hi && (key >= lo || key < sinks);
}

// ------------------------------------------------------------- type traits
template <typename T>
struct Half2;
template <>
struct Half2<__nv_bfloat16> {
  // P = 2^(s - m + kShift).  The running maximum m moves only where a score is
  // above it by more than kSlack, so P <= 2^(kSlack + kShift): bf16 has
  // float32's range.
  static constexpr float kShift = 0.0f, kSlack = 8.0f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
  }
  // u * 0 + acc in both halves
  static __device__ __forceinline__ uint32_t fma0(uint32_t u, uint32_t acc) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(u), "r"(0u), "r"(acc));
    return r;
  }
  // whether either half is an infinity or NaN
  static __device__ __forceinline__ uint32_t bad(uint32_t u) {
    return ((u & 0x7F80u) == 0x7F80u ? 0xFFFFu : 0u) | ((u & 0x7F800000u) == 0x7F800000u ? 0xFFFF0000u : 0u);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct Half2<__half> {
  // P <= 2^12; the shift keeps weights down to 2^-32 of the largest (2^-24
  // without it), which thousands of small ones can add up to.
  static constexpr float kShift = 8.0f, kSlack = 4.0f;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&u));
  }
  static __device__ __forceinline__ uint32_t fma0(uint32_t u, uint32_t acc) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(u), "r"(0u), "r"(acc));
    return r;
  }
  static __device__ __forceinline__ uint32_t bad(uint32_t u) {
    return ((u & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u) | ((u & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u);
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// An 8 x 8 matrix of 16-bit values over the warp (row lane / 4, columns
// 2 (lane % 4), + 1), transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t u) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(u));
  return r;
}
// 16 bytes global -> shared, zeros where !live (nothing is read then).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool live) {
  const int bytes = live ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// --------------------------------------------------------------- few rows
// Warps of a CTA and stages of each warp's ring.  A warp's step is a chain of
// latencies (products, shuffles, exponentials), so warps count for more than
// copies far ahead.  16 sessions x 8 key heads x 8208 keys of 128, in one series
// of runs: six warps of two stages, two CTAs an SM (102 KB each), 80.6 us; four
// of three 81.5; four of two (three CTAs) 87.2; eight of two 87.6.  17 to 32 rows
// of heads of 128 (254 registers a thread, 116 KB) leave room for one CTA alone.
constexpr int kRowsWarps = 6;
constexpr int kRowsStages = 2;
constexpr int kRowsMaxCluster = 8;

struct RowsParams {
  const void *q, *k, *v;
  void *out;
  long long qs[3], ks[3], vs[3], os[3];  // strides of batch, head, token (pages: page, head, token)
  const int32_t *kv_lens;                // nullptr: every session has lk keys
  const int32_t *block_table;            // [B, max_pages] (paged)
  float *part;                           // partial results (n_split > kRowsMaxCluster), else nullptr
  WindowRule rule;
  int B, Hq, Hk, Lq, lk;                 // lk: keys a session can have
  int page, max_pages, n_pages;
  int group, rows, row_tiles;            // rows = group * Lq of one key head
  int n_split;
  int same_strides;                      // k and v have the same
  FastDiv by_split, by_tiles, by_hk, by_group, by_page;
  float scale_log2;
};

// One CTA: a tile of rows of one (session, key head), part `split` of their
// virtual keys.  Each of its warps takes every kRowsWarps-th group of 16 keys
// through a ring of its own in shared memory (cp.async, no CTA barrier in the
// loop).  The products are m16n8k16 ones whose rows are the query heads that
// share the key head, so a key is read once for all of them: S = Q K^T and
// O += P V over 16 MT rows, or, for at most 8 rows (MT 0, most single tokens),
// S^T = K Q^T and O^T += V^T P^T, half as many products.  The warps' results
// are joined in shared memory, the CTAs' through distributed shared memory of
// a cluster, or, for more parts than a cluster has, from `part` by
// window_rows_join_kernel.  The order of every sum is fixed.
//
// Bound: HBM, each key and value once, where there are keys enough: 16 sessions
// of 8 key heads, 8208 keys of 128 in pages of 64, 83.5 us = 6.3 TB/s (0.97 of
// the measured copy); small calls by latency: 24 heads, 1088 keys, 8.2 us; 17 to
// 32 rows of heads of 128 by the one CTA an SM: 28 query and 4 key heads,
// 8 queries over 30000 keys, 50 us = 1.2 TB/s.
// mma.sync serves here: with 16 rows or fewer the products are a tenth of the
// time, and their operands go through registers with no descriptor or TMEM
// traffic.
template <typename T, int D, int MT, bool kPaged>
struct RowsSmem {
  static constexpr int row_bytes = D * 2;
  static constexpr int group_bytes = 16 * row_bytes;               // 16 keys of K or V
  static constexpr int warp_bytes = kRowsStages * 2 * group_bytes;
  static constexpr int ring = kRowsWarps * warp_bytes;
  static constexpr int rows = MT == 0 ? 8 : 16 * MT;
  static constexpr int join = kRowsWarps * rows * (D + 4) * 4;                  // O, m, l of each warp
  static constexpr int bytes = (ring > join ? ring : join) + rows * (D + 4) * 4;  // + the CTA's box
};

// Where a value of a virtual key lies (nullptr: its page is not one).
template <typename T, bool kPaged>
__device__ __forceinline__ const T *rows_value(const RowsParams &p, int b, int hk, int key) {
  const T *v = static_cast<const T *>(p.v) + hk * p.vs[1];
  if (!kPaged) return v + b * p.vs[0] + key * p.vs[2];
  const int pg = __ldg(p.block_table + (long long)b * p.max_pages + key / p.page);
  return pg < 0 || pg >= p.n_pages ? nullptr : v + pg * p.vs[0] + (key % p.page) * p.vs[2];
}

// Gives columns c .. c + 3 of a token's row the infinities and NaN of the
// values that it sees and not every row of its tile does.
template <typename T, bool kPaged>
__device__ __noinline__ void rows_give_back(const RowsParams &p, const WindowSpan &span, int b, int hk, int token, int c,
                                            float (&a)[4]) {
  const int pos = span.len - p.Lq + token;
  if (pos < 0) return;
  int lo, hi;
  window_bounds(p.rule, span.len, pos, lo, hi);
  for (int v = 0; v < span.n; ++v) {
    const int key = span.key(v);
    if (!span.some(key) || !window_sees(key, lo, hi, span.sinks)) continue;
    const T *src = rows_value<T, kPaged>(p, b, hk, key);
    if (!src) continue;
    for (int i = 0; i < 4; ++i) {
      const float y = (float)src[c + i];
      if (!isfinite(y)) a[i] += y;
    }
  }
}

// Writes columns c .. c + 3 of row r (token r / group, head r % group).
template <typename T>
__device__ __forceinline__ void rows_store(const RowsParams &p, int b, int hk, int r, int c, const float (&a)[4]) {
  const int token = p.by_group.div(r), head = hk * p.group + r - token * p.group;
  T *dst = static_cast<T *>(p.out) + b * p.os[0] + (long long)head * p.os[1] + (long long)token * p.os[2] + c;
  *reinterpret_cast<uint2 *>(dst) = make_uint2(Half2<T>::pack(a[0], a[1]), Half2<T>::pack(a[2], a[3]));
}

// Joins the parts' (O, m, l) of rows first, first + step, ... of a tile's
// n_rows, normalises and writes them; part(r, j) is the j-th part's row: O, m,
// l and whether the part took an infinity or NaN out of a value that only some
// rows see.
template <typename T, int D, int MT, bool kPaged, typename Part>
__device__ __forceinline__ void window_write(const RowsParams &p, const WindowSpan &span, int b, int hk, int r0,
                                             int n_rows, int first, int step, const Part &part, int thread,
                                             int threads) {
  const int mine = first < n_rows ? (n_rows - first + step - 1) / step : 0;
  for (int x = thread; x < mine * (D / 4); x += threads) {
    const int r = first + x / (D / 4) * step, c = (x % (D / 4)) * 4;
    float m = -INFINITY, bad = 0.0f;
    for (int j = 0; j < p.n_split; ++j) m = fmaxf(m, part(r, j)[D]);
    float l = 0.0f, a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int j = 0; j < p.n_split; ++j) {
      const float *row = part(r, j);
      const float4 tail = *reinterpret_cast<const float4 *>(row + D);
      const float f = tail.x == -INFINITY ? 0.0f : fast_exp2(tail.x - m);
      const float4 v = *reinterpret_cast<const float4 *>(row + c);
      l = fmaf(tail.y, f, l);
      a[0] = fmaf(v.x, f, a[0]), a[1] = fmaf(v.y, f, a[1]), a[2] = fmaf(v.z, f, a[2]), a[3] = fmaf(v.w, f, a[3]);
      if (__float_as_int(tail.z)) bad = 1.0f;
    }
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;  // (a NaN sum stays one)
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] *= inv;
    if (__builtin_expect(bad != 0.0f, 0)) {
      float z[4] = {a[0], a[1], a[2], a[3]};
      rows_give_back<T, kPaged>(p, span, b, hk, p.by_group.div(r0 + r), c, z);
      for (int i = 0; i < 4; ++i) a[i] = z[i];
    }
    rows_store<T>(p, b, hk, r0 + r, c, a);
  }
}

template <typename T, int D, int MT, bool kPaged>
__global__ void __launch_bounds__(kRowsWarps * 32) window_rows_kernel(const __grid_constant__ RowsParams p) {
  using S = RowsSmem<T, D, MT, kPaged>;
  using H2 = Half2<T>;
  constexpr int kChunks = D / 8;  // 16-byte pieces of a row
  constexpr int R = S::rows;
  constexpr bool kSwap = MT == 0;
  constexpr int M = kSwap ? 1 : MT;
  extern __shared__ __align__(1024) uint8_t smem_rows[];
  __shared__ int flag_bad;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = p.by_split.div(blockIdx.x), split = blockIdx.x - item * p.n_split;
  const int bh = p.by_tiles.div(item), rt = item - bh * p.row_tiles;
  const int b = p.by_hk.div(bh), hk = bh - b * p.Hk;
  const int r0 = rt * R;  // first row: token r / group, head r % group
  const int r_end = min(p.rows, r0 + R);
  int len = p.kv_lens ? p.kv_lens[b] : p.lk;
  if (len < 0 || len > p.lk) {  // a session longer than its cache: nothing past the cache is read
    if (threadIdx.x == 0) atomicExch(&g_cast_device_error, (int)CAST_ERR_INVALID_ARGUMENT);
    len = min(max(len, 0), p.lk);
  }
  const WindowSpan span = window_span(p.rule, len, p.Lq, p.by_group.div(r0), p.by_group.div(r_end - 1));
  const int groups = (span.n + 15) / 16;
  // this CTA's groups of 16 keys: an equal share, the first ones one more
  const int share = p.by_split.div(groups), more = groups - share * p.n_split;
  const int g_lo = split * share + min(split, more), g_hi = g_lo + share + (split < more ? 1 : 0);
  const bool partial = span.lo0 != span.lo1 || span.hi0 != span.hi1 || span.unplaced;
  if (threadIdx.x == 0) flag_bad = 0;
  if (p.n_split > 1 && !p.part) cluster_arrive();  // (waited for before the first push)
  __syncthreads();

  // ---- Q fragments: row r = lane / 4 (+ 8), columns 2 (lane % 4) (+ 8) of each 16
  // (kSwap: as the second operand, row lane / 4 alone)
  uint32_t qf[M][D / 16][kSwap ? 2 : 4];
#pragma unroll
  for (int mt = 0; mt < M; ++mt) {
#pragma unroll
    for (int hh = 0; hh < (kSwap ? 1 : 2); ++hh) {
      const int r = r0 + 16 * mt + lane / 4 + 8 * hh;
      const bool on = r < r_end;
      const int i = p.by_group.div(r), g = r - i * p.group;
      const T *src = static_cast<const T *>(p.q) + b * p.qs[0] + (long long)(hk * p.group + g) * p.qs[1] + (long long)i * p.qs[2];
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        qf[mt][s][hh] = on ? *reinterpret_cast<const uint32_t *>(src + 16 * s + 2 * (lane % 4)) : 0u;
        qf[mt][s][(kSwap ? 1 : 2) + hh] = on ? *reinterpret_cast<const uint32_t *>(src + 16 * s + 8 + 2 * (lane % 4)) : 0u;
      }
    }
  }
  // The two rows of each product tile whose scores this lane holds, and what they see.
  auto own_row = [&](int mt, int hh) { return kSwap ? 2 * (lane % 4) + hh : 16 * mt + lane / 4 + 8 * hh; };
  int lo[M][2], hi[M][2];
#pragma unroll
  for (int mt = 0; mt < M; ++mt)
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      const int r = r0 + own_row(mt, hh);
      const int pos = len - p.Lq + p.by_group.div(r);
      lo[mt][hh] = hi[mt][hh] = 0;
      if (r < r_end && pos >= 0) window_bounds(p.rule, len, pos, lo[mt][hh], hi[mt][hh]);
    }

  // O: [16 rows][8 columns] tiles, or (kSwap) [16 columns][8 rows] ones
  constexpr int kOut = kSwap ? D / 16 : D / 8;
  float o[M][kOut][4];
  float m_run[M][2], l_run[M][2];
#pragma unroll
  for (int mt = 0; mt < M; ++mt) {
#pragma unroll
    for (int j = 0; j < kOut; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[mt][j][c] = 0.0f;
    m_run[mt][0] = m_run[mt][1] = -INFINITY;
    l_run[mt][0] = l_run[mt][1] = 0.0f;
  }

  const uint32_t ring = castdev::smem_u32(smem_rows) + warp * S::warp_bytes;
  const T *kbase = static_cast<const T *>(p.k) + (kPaged ? 0 : b * p.ks[0]) + hk * p.ks[1];
  const T *vbase = static_cast<const T *>(p.v) + (kPaged ? 0 : b * p.vs[0]) + hk * p.vs[1];

  // Where key lane % 16 of group g lies (nullptr: no key there).  A lane works
  // out one key, a group ahead, and its row's copies take the pointer from it.
  struct Place {
    const T *k, *v;
  };
  auto place_of = [&](int g) -> Place {
    Place at{nullptr, nullptr};
    const int v = 16 * g + (lane & 15);
    if (g >= g_hi || v >= span.n) return at;
    const int key = span.key(v);
    long long ko, vo;
    if (kPaged) {
      const int pg_at = p.by_page.div(key), in = key - pg_at * p.page;
      const int pg = __ldg(p.block_table + (long long)b * p.max_pages + pg_at);
      if (pg < 0 || pg >= p.n_pages) {
        atomicExch(&g_cast_device_error, (int)CAST_ERR_INVALID_ARGUMENT);
        return at;
      }
      ko = pg * p.ks[0] + in * p.ks[2];
      vo = p.same_strides ? ko : pg * p.vs[0] + in * p.vs[2];
    } else {
      ko = key * p.ks[2];
      vo = p.same_strides ? ko : key * p.vs[2];
    }
    at.k = kbase + ko;
    at.v = vbase + vo;
    return at;
  };
  // Starts the copies of a group into stage st; returns a bit for each of the
  // 16 keys that are there.
  const ptrdiff_t v_from_k = reinterpret_cast<const char *>(vbase) - reinterpret_cast<const char *>(kbase);
  auto start = [&](int st, const Place &at) -> uint32_t {
    const uint32_t there = __ballot_sync(0xffffffffu, at.k != nullptr) & 0xFFFFu;
    const uint32_t dst = ring + st * 2 * S::group_bytes;
    constexpr int kRowsPer = 32 / kChunks;  // rows a pass of the warp covers
    const int c = lane % kChunks;
    const unsigned long long mine = reinterpret_cast<unsigned long long>(at.k ? at.k : kbase);
    const unsigned long long mine_v = reinterpret_cast<unsigned long long>(at.k ? at.v : vbase);
#pragma unroll
    for (int i = 0; i < 16 / kRowsPer; ++i) {
      const int row = i * kRowsPer + lane / kChunks;
      const bool live = (there >> row) & 1u;
      const char *kr = reinterpret_cast<const char *>(__shfl_sync(0xffffffffu, mine, row)) + 16 * c;
      const char *vr = p.same_strides ? kr + v_from_k
                                      : reinterpret_cast<const char *>(__shfl_sync(0xffffffffu, mine_v, row)) + 16 * c;
      const uint32_t off = row * S::row_bytes + ((c ^ (row & 7)) * 16);
      cp_async16(dst + off, kr, live);
      cp_async16(dst + S::group_bytes + off, vr, live);
    }
    return there;
  };

  // groups g_lo + warp + kRowsWarps * t of this warp
  const int first = g_lo + warp;
  uint32_t there[kRowsStages];
  Place next = place_of(first);
#pragma unroll
  for (int st = 0; st < kRowsStages - 1; ++st) {
    const Place at = next;
    next = place_of(first + kRowsWarps * (st + 1));
    there[st] = start(st, at);
    cp_async_commit();
  }
  there[kRowsStages - 1] = 0;
  int saw_bad = 0;

  for (int t = 0; first + kRowsWarps * t < g_hi; ++t) {
    const int g = first + kRowsWarps * t;
    const int st = t % kRowsStages;
    cp_async_wait<kRowsStages - 2>();
    __syncwarp();
    {  // the stage read in the last step is free: start the group it takes
      const int sn = (t + kRowsStages - 1) % kRowsStages;
      const Place at = next;
      next = place_of(g + kRowsWarps * kRowsStages);
      const uint32_t bits = start(sn, at);
      cp_async_commit();
#pragma unroll
      for (int x = 0; x < kRowsStages; ++x)
        if (x == sn) there[x] = bits;
    }
    uint32_t mine = 0;
#pragma unroll
    for (int x = 0; x < kRowsStages; ++x)
      if (x == st) mine = there[x];
    const uint32_t ks = ring + st * 2 * S::group_bytes, vs = ks + S::group_bytes;

    // S = Q K^T of 16 keys; s[mt][..][..]: this lane's two rows by four keys
    float s[M][2][4];
#pragma unroll
    for (int mt = 0; mt < M; ++mt)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[mt][0][c] = s[mt][1][c] = 0.0f;
    if constexpr (kSwap) {  // S^T = K Q^T, two chains over the columns
      const int row = (lane & 7) + (((lane >> 3) & 1) << 3), cc = lane >> 4;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t kf[4];
        ldmatrix_x4(ks + row * S::row_bytes + (((2 * j + cc) ^ (row & 7)) * 16), kf);
        H2::mma(s[0][j & 1], kf, qf[0][j][0], qf[0][j][1]);
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) s[0][0][c] += s[0][1][c];
    } else {
      const int row = (lane & 7) + ((lane >> 4) << 3), cc = (lane >> 3) & 1;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t kf[4];
        ldmatrix_x4(ks + row * S::row_bytes + (((2 * j + cc) ^ (row & 7)) * 16), kf);
#pragma unroll
        for (int mt = 0; mt < M; ++mt) {
          H2::mma(s[mt][0], qf[mt][j], kf[0], kf[1]);
          H2::mma(s[mt][1], qf[mt][j], kf[2], kf[3]);
        }
      }
    }
    // Whether every row sees every key of the group (sinks and window never
    // share one then).
    const int k_first = span.key(16 * g), k_last = span.key(16 * g + 15);
    const bool whole = mine == 0xFFFFu && !span.unplaced && k_last - k_first == 15 &&
                       (k_last < min(span.sinks, span.hi0) || (k_first >= span.lo1 && k_last < span.hi0));
    // This lane's keys: 2 (lane % 4) + {0, 1, 8, 9}, or (kSwap) lane / 4 + {0, 8}.
    constexpr int kKeys = kSwap ? 2 : 4;
    auto score = [&](int mt, int hh, int c) -> float & {
      return kSwap ? s[0][0][2 * c + hh] : s[mt][c >> 1][2 * hh + (c & 1)];
    };
    int key[kKeys];
    uint32_t col_there = 0;
#pragma unroll
    for (int c = 0; c < kKeys; ++c) {
      const int col = kSwap ? lane / 4 + 8 * c : 2 * (lane % 4) + (c & 1) + 8 * (c >> 1);
      key[c] = span.key(16 * g + col);
      if ((mine >> col) & 1u) col_there |= 1u << c;
    }
    uint32_t pf[M][4];  // (kSwap: [0][0..1])
#pragma unroll
    for (int mt = 0; mt < M; ++mt) {
      float mx[2];
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        float x = -INFINITY;
#pragma unroll
        for (int c = 0; c < kKeys; ++c) {
          float &v = score(mt, hh, c);
          const bool on = whole || (((col_there >> c) & 1u) && window_sees(key[c], lo[mt][hh], hi[mt][hh], span.sinks) &&
                                    hi[mt][hh] > 0);
          v = on ? v * p.scale_log2 : -INFINITY;
          x = fmaxf(x, v);
        }
        mx[hh] = x;
      }
#pragma unroll
      for (int d = kSwap ? 4 : 1; d <= (kSwap ? 16 : 2); d *= 2) {
        mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], d));
        mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], d));
      }
      const bool move0 = mx[0] > m_run[mt][0] + H2::kSlack, move1 = mx[1] > m_run[mt][1] + H2::kSlack;
      if (__any_sync(0xffffffffu, move0 || move1)) {
        const float n0 = move0 ? mx[0] : m_run[mt][0], n1 = move1 ? mx[1] : m_run[mt][1];
        const float f0 = move0 ? fast_exp2(m_run[mt][0] - n0) : 1.0f, f1 = move1 ? fast_exp2(m_run[mt][1] - n1) : 1.0f;
        m_run[mt][0] = n0, m_run[mt][1] = n1;
        l_run[mt][0] *= f0, l_run[mt][1] *= f1;
#pragma unroll
        for (int j = 0; j < kOut; ++j) {
          o[mt][j][0] *= f0, o[mt][j][1] *= kSwap ? f1 : f0;
          o[mt][j][2] *= kSwap ? f0 : f1, o[mt][j][3] *= f1;
        }
      }
      // (the sums take the weights that P V uses, so that these sum to one)
      const float base0 = m_run[mt][0] == -INFINITY ? 0.0f : m_run[mt][0] - H2::kShift;
      const float base1 = m_run[mt][1] == -INFINITY ? 0.0f : m_run[mt][1] - H2::kShift;
      if constexpr (kSwap) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t u = H2::pack(fast_exp2(score(0, 0, c) - base0), fast_exp2(score(0, 1, c) - base1));
          pf[0][c] = transpose8(u);
          const float2 w = H2::unpack(u);
          l_run[0][0] += w.x;
          l_run[0][1] += w.y;
        }
      } else {
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            const float base = hh == 0 ? base0 : base1;
            const uint32_t u = H2::pack(fast_exp2(s[mt][nt][2 * hh] - base), fast_exp2(s[mt][nt][2 * hh + 1] - base));
            pf[mt][2 * nt + hh] = u;
            const float2 w = H2::unpack(u);
            l_run[mt][hh] += w.x + w.y;
          }
      }
    }
    if (partial && !whole) {
      // A key that only some rows of the tile see: its value meets a zero
      // weight in the others, so an infinity or NaN there is taken out here
      // and given back to the rows that see it at the end.
      const int col = lane & 15;
      const int kk = span.key(16 * g + col);
      const bool some = ((mine >> col) & 1u) && span.some(kk);
      uint32_t todo = __ballot_sync(0xffffffffu, some) & 0xFFFFu;
      while (todo) {
        const int row = __ffs(todo) - 1;
        todo &= todo - 1;
        uint32_t *w = reinterpret_cast<uint32_t *>(smem_rows + (vs - castdev::smem_u32(smem_rows)) + row * S::row_bytes);
#pragma unroll
        for (int x = lane; x < D / 2; x += 32) {
          const uint32_t u = w[x], bad = H2::bad(u);
          if (bad) {
            w[x] = u & ~bad;
            saw_bad = 1;
          }
        }
      }
      __syncwarp();
    }
    // O += P V
    if constexpr (kSwap) {  // O^T += V^T P^T
      const int row = (lane & 7) + ((lane >> 4) << 3), cc = (lane >> 3) & 1;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t vf[4];
        ldmatrix_x4_trans(vs + row * S::row_bytes + (((2 * j + cc) ^ (row & 7)) * 16), vf);
        H2::mma(o[0][j], vf, pf[0][0], pf[0][1]);
      }
    } else {
      const int row = (lane & 7) + (((lane >> 3) & 1) << 3), cc = lane >> 4;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t vf[4];
        ldmatrix_x4_trans(vs + row * S::row_bytes + (((2 * j + cc) ^ (row & 7)) * 16), vf);
#pragma unroll
        for (int mt = 0; mt < M; ++mt) {
          H2::mma(o[mt][2 * j], pf[mt], vf[0], vf[1]);
          H2::mma(o[mt][2 * j + 1], pf[mt], vf[2], vf[3]);
        }
      }
    }
    __syncwarp();
  }
  cp_async_wait<0>();
  if (saw_bad) flag_bad = 1;
  __syncthreads();

  // ---- join the warps: (O, m, l) of each row in shared memory, rows of D + 4 floats
  constexpr int kRow = D + 4;
  const int n_rows = r_end - r0;
  float *js = reinterpret_cast<float *>(smem_rows);
  float *box = reinterpret_cast<float *>(smem_rows + (S::ring > S::join ? S::ring : S::join));
#pragma unroll
  for (int mt = 0; mt < M; ++mt)
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      float l = l_run[mt][hh];
#pragma unroll
      for (int d = kSwap ? 4 : 1; d <= (kSwap ? 16 : 2); d *= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
      const int r = own_row(mt, hh);
      if (r >= n_rows) continue;
      float *row = js + (warp * R + r) * kRow;
      if constexpr (kSwap) {
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          row[16 * j + lane / 4] = o[0][j][hh];
          row[16 * j + lane / 4 + 8] = o[0][j][2 + hh];
        }
      } else {
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
          *reinterpret_cast<float2 *>(row + 8 * j + 2 * (lane % 4)) = make_float2(o[mt][j][2 * hh], o[mt][j][2 * hh + 1]);
      }
      if (kSwap ? lane < 4 : lane % 4 == 0) {
        row[D] = m_run[mt][hh];
        row[D + 1] = l;
      }
    }
  __syncthreads();
  // Row r of every CTA of the cluster goes to CTA r % n_split, place
  // (r / n_split) n_split + split of its box (R rows in all), which
  // joins them: one barrier between the pushes and the joins, and nobody's
  // memory is touched after it.
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const bool push = p.n_split > 1 && !p.part;
  if (push) cluster_wait();  // every CTA of the cluster runs
  for (int x = threadIdx.x; x < n_rows * (D / 4); x += blockDim.x) {
    const int r = x / (D / 4), c = (x % (D / 4)) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) m = fmaxf(m, js[(w * R + r) * kRow + D]);
    float l = 0.0f;
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) {
      const float *row = js + (w * R + r) * kRow;
      const float f = row[D] == -INFINITY ? 0.0f : fast_exp2(row[D] - m);
      const float4 v = *reinterpret_cast<const float4 *>(row + c);
      l = fmaf(row[D + 1], f, l);
      a.x = fmaf(v.x, f, a.x), a.y = fmaf(v.y, f, a.y), a.z = fmaf(v.z, f, a.z), a.w = fmaf(v.w, f, a.w);
    }
    float *dst = push ? cluster.map_shared_rank(box, r % p.n_split) + (r / p.n_split * p.n_split + split) * kRow
                      : (p.part ? p.part + (long long)blockIdx.x * (R * kRow) : box) + r * kRow;
    *reinterpret_cast<float4 *>(dst + c) = a;
    if (c == 0) *reinterpret_cast<float4 *>(dst + D) = make_float4(m, l, __int_as_float(flag_bad), 0.0f);
  }
  if (p.part) return;  // window_rows_join_kernel joins the CTAs
  if (push) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  window_write<T, D, MT, kPaged>(p, span, b, hk, r0, n_rows, push ? split : 0, push ? p.n_split : 1,
                                 [&](int r, int j) { return box + (push ? r / p.n_split * p.n_split + j : r) * kRow; },
                                 (int)threadIdx.x, (int)blockDim.x);
}

// Joins the parts that window_rows_kernel left in p.part: one CTA for a row
// of a tile.  Its threads take the parts' maxima and sums side by side, then
// every kRowsJoin-th part's O, so that no load waits for another (a thread
// walking the parts one after the other took 20 us for 37 parts).
constexpr int kRowsJoin = 8;
template <typename T, int D, int MT, bool kPaged>
__global__ void __launch_bounds__(kRowsJoin * D / 4) window_rows_join_kernel(const __grid_constant__ RowsParams p) {
  constexpr int R = RowsSmem<T, D, MT, kPaged>::rows, kRow = D + 4, kThreads = kRowsJoin * D / 4;
  __shared__ float4 acc_s[kRowsJoin][D / 4];
  __shared__ float max_s[kThreads / 32], sum_s[kRowsJoin];
  const int item = blockIdx.x / R, r = blockIdx.x % R;
  const int bh = p.by_tiles.div(item), rt = item - bh * p.row_tiles;
  const int b = p.by_hk.div(bh), hk = bh - b * p.Hk;
  const int r0 = rt * R, r_end = min(p.rows, r0 + R);
  if (r0 + r >= r_end) return;  // (whole CTAs)
  const float *base = p.part + (long long)item * p.n_split * (R * kRow) + r * kRow;
  auto part = [&](int j) { return base + (long long)j * (R * kRow); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the parts' maximum
  float m = -INFINITY;
  for (int j = threadIdx.x; j < p.n_split; j += kThreads) m = fmaxf(m, part(j)[D]);
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (lane == 0) max_s[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) m = fmaxf(m, max_s[w]);
  // sums and O
  const int g = threadIdx.x / (D / 4), c = threadIdx.x % (D / 4);
  float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f;
  bool bad = false;
#pragma unroll 4
  for (int j = g; j < p.n_split; j += kRowsJoin) {
    const float4 tail = *reinterpret_cast<const float4 *>(part(j) + D);
    const float4 v = *reinterpret_cast<const float4 *>(part(j) + 4 * c);
    const float f = tail.x == -INFINITY ? 0.0f : fast_exp2(tail.x - m);
    l = fmaf(tail.y, f, l);
    a.x = fmaf(v.x, f, a.x), a.y = fmaf(v.y, f, a.y), a.z = fmaf(v.z, f, a.z), a.w = fmaf(v.w, f, a.w);
    bad = bad || __float_as_int(tail.z) != 0;
  }
  acc_s[g][c] = a;
  if (c == 0) sum_s[g] = l;
  const bool any_bad = __syncthreads_or(bad);
  if (g != 0) return;
  float y[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  l = 0.0f;
#pragma unroll
  for (int j = 0; j < kRowsJoin; ++j) {
    const float4 v = acc_s[j][c];
    y[0] += v.x, y[1] += v.y, y[2] += v.z, y[3] += v.w;
    l += sum_s[j];
  }
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;  // (a NaN sum stays one)
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] *= inv;
  if (any_bad) {
    const int len = min(max(p.kv_lens ? p.kv_lens[b] : p.lk, 0), p.lk);
    const WindowSpan span = window_span(p.rule, len, p.Lq, p.by_group.div(r0), p.by_group.div(r_end - 1));
    rows_give_back<T, kPaged>(p, span, b, hk, p.by_group.div(r0 + r), 4 * c, y);
  }
  rows_store<T>(p, b, hk, r0 + r, 4 * c, y);
}

}  // namespace castk
