// Rotary positions, and the RMS norm of query and key heads with the rotation
// in the same pass.
//
// A head vector x of D values becomes, with r = 1 (no norm) or
// r = 1 / sqrt(mean(x^2) + eps) and weight w,
//   z_i = x_i * r * w_i,
//   (y_a, y_b) = (z_a c - z_b s, z_a s + z_b c)   for each pair p of the first R values,
// where (a, b) is (2p, 2p + 1) in the interleaved layout and (p, p + R/2) in
// the half layout, and (c, s) is row `position` of a float32 table: its angles
// are formed in 64 bits when the table is made, since a float32 angle of a far
// position has lost the turn's fraction.  Norm, rotation and sums are float32;
// the result is rounded to the output type once.
//
// Bound: HBM, if instructions do not come first.  Every value is read and
// written once, in 16-byte pieces of eight values (two for float32), and a head
// is a group of 4 to 32 lanes of one warp, so its sum of squares is a shuffle
// reduction.  A lane has two pieces, half a head apart, where it can (the pairs
// of the half layout are then its own), else one, and a partner's values are a
// shuffle away.  No shared memory.
// A lane keeps the same columns for every head of its token, so the table row
// is read once per token and lane and its (c, s) stay in registers; a few heads
// are loaded before the first is worked on.
//
// Measured (B200, graph over rotating inputs): rotation alone, 31680 tokens of
// 24 heads of 128 bf16, 66 us = 5.9 TB/s, 0.90 of the measured copy; 12500 in
// float32 55 us = 5.6 TB/s, 0.85; with the norm, 3520 tokens of 24 + 24 heads,
// 24.1 us = 3.6 TB/s, 0.55: about 200 instructions a head and 16 lanes (58 % of
// the issue slots), where the rotation alone takes 150 (half of it position
// and table row).  The norm's kernels spill: a head's values, the weight in
// pairs, (cos, sin) and 64-bit pointers are more than the 64 or 72 registers
// below.  Bytes stored / loaded a thread: one piece, pairs side by side,
// 16-bit 190 / 190 and float32 380 / 280; half layout 330 / 220 and 540 / 550;
// two pieces 1000 / 500 and 1400 to 1700 / 1000 to 1400.
#pragma once

#include <cuda_fp16.h>

#include "attention.cuh"
#include "common.cuh"
#include "compact.cuh"

namespace castk {

__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

constexpr int kRotaryThreads = 128;
constexpr int kRotaryRun = 4;  // tokens a lane takes one after the other
// Heads in flight per lane of one piece or two, and CTAs on an SM.  Under the
// norm both counts spill (see above), and these are the best of the counts
// tried, not the best there could be without spills (one piece: 4 heads and
// 6 CTAs are level; two pieces: 3 heads and 6 CTAs take 94 us where 2 and 7
// take 69).
constexpr int rotary_batch(int pieces) { return pieces == 2 ? 2 : 3; }
constexpr int rotary_ctas(int pieces) { return pieces == 2 ? 7 : 8; }

// One tensor of a call: q, k and (copied only) v.
struct RotaryTensor {
  const void *src;
  void *dst;
  const void *weight;  // nullptr: no norm
  long long ss[3];     // source strides of batch, token, head (elements)
  long long ds[3];     // destination strides
  int heads;
};

struct RotaryParams {
  RotaryTensor t[3];
  const float *table;  // [table_rows, R/2] (cos, sin)
  const void *positions;
  const void *slots;  // paged destination of tensors 1 and 2 (nullptr: strides)
  long long pos_batch_stride, first_position;
  long long n_slots;
  int table_rows, pos64, slots64, n_axes, axis_end0, axis_end1;
  int page;
  int B, L, D, R;
  int pieces, lanes;                // of eight values to a lane (1 or 2); lanes of one head
  int slots_per_token, slots_log2;  // heads of one token at once, a power of two
  int tokens_per_cta;
  int inverse, weight_f32, weight_per_head;
  float eps, inv_d;
};

// Eight consecutive values as loaded, and their float32 values.
template <typename T>
struct Eight {
  uint4 w = {};
  __device__ __forceinline__ void load(const T *p) { w = *reinterpret_cast<const uint4 *>(p); }
  __device__ __forceinline__ void values(float (&x)[8]) const;
};
template <>
__device__ __forceinline__ void Eight<__nv_bfloat16>::values(float (&x)[8]) const {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(u[i] << 16);
    x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
  }
}
template <>
__device__ __forceinline__ void Eight<__half>::values(float (&x)[8]) const {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <>
struct Eight<float> {
  float4 a = {}, b = {};
  __device__ __forceinline__ void load(const float *p) {
    a = *reinterpret_cast<const float4 *>(p);
    b = *reinterpret_cast<const float4 *>(p + 4);
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
    x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
};

__device__ __forceinline__ void store8(__nv_bfloat16 *p, const float (&x)[8]) {
  *reinterpret_cast<uint4 *>(p) = to_bf16x8(x);
}
__device__ __forceinline__ void store8(__half *p, const float (&x)[8]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    u[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  *reinterpret_cast<uint4 *>(p) = make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ void store8(float *p, const float (&x)[8]) {
  *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4 *>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}

__device__ __forceinline__ long long load_index(const void *p, int is64, long long i) {
  return is64 ? __ldg(static_cast<const long long *>(p) + i)
              : (long long)__ldg(static_cast<const int32_t *>(p) + i);
}

// A lane's columns of a head: kC pieces of eight, 8 c and, with two, D / 2 + 8 c
// (which then holds the other values of its pairs in the half layout).
template <typename InT, typename OutT, bool kNorm, bool kHalf, int kC, int kLanes>
struct RotaryLane {
  static constexpr int kBatch = rotary_batch(kC);
  static constexpr int kPairs = kHalf ? 8 : 4 * kC;  // table entries of a lane's columns
  float cs[kPairs], sn[kPairs];
  bool live, turns[kC];
  bool blank;  // (without the norm) this token's position is unknown: it is read as zeros
  int c, h0, step, partner, second;  // second: columns from the first piece to the second

  template <bool kBlank>
  __device__ __forceinline__ void load(const RotaryParams &p, const RotaryTensor &t, const InT *row, int hb,
                                       Eight<InT> (&raw)[kBatch][kC]) const {
    const InT *src = row + (long long)(hb + h0) * t.ss[2];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (live && hb + u * step + h0 < t.heads) {
#pragma unroll
        for (int j = 0; j < kC; ++j) raw[u][j].load(src + j * second);
      }
      src += step * t.ss[2];
    }
    if (kBlank && blank) clear(raw);
  }
  __device__ __forceinline__ void clear(Eight<InT> (&raw)[kBatch][kC]) const {
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
#pragma unroll
      for (int j = 0; j < kC; ++j) raw[u][j] = Eight<InT>{};
  }
  // Zeros in place of a tensor's heads.
  __device__ __forceinline__ void zeros(const RotaryTensor &t, OutT *at, long long at_step) const {
    const float x[8] = {};
#pragma unroll 1
    for (int h = h0; live && h < t.heads; h += step)
#pragma unroll
      for (int j = 0; j < kC; ++j) store8(at + h * at_step + j * second, x);
  }

  // One tensor's heads of one token, h0, h0 + step, ... below t.heads.  kTurn:
  // norm and rotate (q and k); at: the destination of head 0, nullptr: nothing
  // is written.
  template <bool kTurn>
  __device__ __forceinline__ void run(const RotaryParams &p, const RotaryTensor &t, const InT *row, OutT *at,
                                      long long at_step, Eight<InT> (&raw)[kBatch][kC]) const {
    uint64_t w[4 * kC];  // the weight's values, in pairs
    auto weight = [&](int h) {
      const long long wo = (p.weight_per_head ? (long long)h * p.D : 0) + 8 * c;
#pragma unroll
      for (int j = 0; j < kC; ++j) {
        float f[8];
        if (p.weight_f32) {
          Eight<float> e;
          e.load(static_cast<const float *>(t.weight) + wo + j * second);
          e.values(f);
        } else {
          Eight<InT> e;
          e.load(static_cast<const InT *>(t.weight) + wo + j * second);
          e.values(f);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) w[4 * j + i] = f2_pack(f[2 * i], f[2 * i + 1]);
      }
    };
    const bool normed = kNorm && kTurn && t.weight != nullptr;
    if (normed && live && !p.weight_per_head) weight(0);
    for (int hb = 0; hb < t.heads; hb += step * kBatch) {  // same trip count in the whole CTA
      if (hb > 0) load<kTurn && !kNorm>(p, t, row, hb, raw);
      OutT *dst = at + (long long)(hb + h0) * at_step;
#pragma unroll
      for (int u = 0; u < kBatch; ++u, dst += step * at_step) {
        const int h = hb + u * step + h0;
        const bool on = live && h < t.heads;
        float x[kC][8];  // (lanes without a head compute what they hold and write nothing)
#pragma unroll
        for (int j = 0; j < kC; ++j) raw[u][j].values(x[j]);
        if (normed) {
          uint64_t sum2 = 0;
#pragma unroll
          for (int j = 0; j < kC; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint64_t v = f2_pack(x[j][2 * i], x[j][2 * i + 1]);
              sum2 = f2_fma(v, v, sum2);
            }
          float lo, hi;
          f2_unpack(sum2, lo, hi);
          float sum = lo + hi;
#pragma unroll
          for (int s = kLanes / 2; s >= 1; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
          const float r = rsqrtf(fmaf(sum, p.inv_d, p.eps));
          const uint64_t r2 = f2_pack(r, r);
          if (p.weight_per_head && on) weight(h);
#pragma unroll
          for (int j = 0; j < kC; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              f2_unpack(f2_mul(f2_mul(f2_pack(x[j][2 * i], x[j][2 * i + 1]), r2), w[4 * j + i]), x[j][2 * i], x[j][2 * i + 1]);
        }
        if constexpr (kTurn && kHalf && kC == 2) {
          if (turns[0]) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float a = x[0][i], q = x[1][i];
              x[0][i] = fmaf(a, cs[i], -(q * sn[i]));
              x[1][i] = fmaf(a, sn[i], q * cs[i]);
            }
          }
        } else if constexpr (kTurn && kHalf) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float o = __shfl_sync(0xffffffffu, x[0][i], partner);
            if (turns[0]) x[0][i] = fmaf(x[0][i], cs[i], o * sn[i]);
          }
        } else if constexpr (kTurn) {
#pragma unroll
          for (int j = 0; j < kC; ++j) {
            if (turns[j]) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float a = x[j][2 * i], q = x[j][2 * i + 1];
                x[j][2 * i] = fmaf(a, cs[4 * j + i], -(q * sn[4 * j + i]));
                x[j][2 * i + 1] = fmaf(a, sn[4 * j + i], q * cs[4 * j + i]);
              }
            }
          }
        }
        if (on && at) {
#pragma unroll
          for (int j = 0; j < kC; ++j) store8(dst + j * second, x[j]);
        }
      }
    }
  }
};

template <typename InT, typename OutT, bool kNorm, bool kHalf, int kC, int kLanes>
__global__ void __launch_bounds__(kRotaryThreads, rotary_ctas(kC)) rotary_kernel(const __grid_constant__ RotaryParams p) {
  RotaryLane<InT, OutT, kNorm, kHalf, kC, kLanes> f;
  constexpr int kPairs = f.kPairs;
  int *err = &g_cast_device_error;
  f.c = threadIdx.x & (kLanes - 1);
  const int c = f.c, group = threadIdx.x / kLanes;
  f.step = p.slots_per_token;  // a power of two
  f.h0 = group & (p.slots_per_token - 1);
  const int b = blockIdx.y + blockIdx.z * gridDim.y;
  if (b >= p.B) return;  // (whole CTAs)
  const int half_pairs = p.R >> 1, half_chunks = p.R >> 4;
  f.second = p.D >> 1;
  // first pair of each piece (two pieces in the half layout have the same pairs)
  const int pair0 = kHalf ? (kC == 2 || c < half_chunks ? 8 * c : 8 * (c - half_chunks)) : 4 * c;
  const bool flip = (p.inverse != 0) != (kHalf && kC == 1 && c < half_chunks);
  f.partner = kHalf && kC == 1 ? (((threadIdx.x & 31) - c + (c < half_chunks ? c + half_chunks : c - half_chunks)) & 31) : 0;

  const InT *src[3];
  OutT *dst[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    src[i] = static_cast<const InT *>(p.t[i].src) + b * p.t[i].ss[0] + 8 * c;
    dst[i] = static_cast<OutT *>(p.t[i].dst) + b * p.t[i].ds[0] + 8 * c;
  }
  Eight<InT> raw[rotary_batch(kC)][kC] = {};  // zeros where a lane has no column: they enter a head's sum
  const int l_end = min(p.L, (int)(blockIdx.x + 1) * p.tokens_per_cta);
  for (int l = blockIdx.x * p.tokens_per_cta + (group >> p.slots_log2);; l += (kRotaryThreads / kLanes) >> p.slots_log2) {
    // the lanes of a warp may have different tokens: it leaves together
    if (!__any_sync(0xffffffffu, l < l_end)) break;
    const bool live_token = l < l_end;
    f.live = live_token && 8 * kC * c < p.D;
    bool any_turns = false;
#pragma unroll
    for (int j = 0; j < kC; ++j) {
      f.turns[j] = f.live && (kHalf && kC == 2 ? p.R > 0 : 8 * c + j * f.second < p.R);
      any_turns = any_turns || f.turns[j];
    }

    // on its way while the position and then its table row are fetched
    f.blank = false;
    f.template load<false>(p, p.t[0], src[0] + l * p.t[0].ss[1], 0, raw);

    // ---- this lane's (cos, sin): none where its columns are not rotated
    if (p.R > 0) {
      int pos[3] = {0, 0, 0};
      bool known = true;  // every position of this token is a row of the table
      if (live_token) {
        if (!p.positions) {
          pos[0] = (int)p.first_position + l;
          known = pos[0] < p.table_rows;
        } else {
          const long long at = b * p.pos_batch_stride + (long long)l * p.n_axes;
#pragma unroll
          for (int a = 0; a < 3; ++a) {
            if (a > 0 && p.n_axes == 1) break;
            if (p.pos64) {
              const long long v = __ldg(static_cast<const long long *>(p.positions) + at + a);
              known = known && v >= 0 && v < p.table_rows;
              pos[a] = (int)v;
            } else {
              pos[a] = __ldg(static_cast<const int32_t *>(p.positions) + at + a);
              known = known && (uint32_t)pos[a] < (uint32_t)p.table_rows;
            }
          }
        }
      }
      if (__any_sync(0xffffffffu, !known)) {
        // Zeros, and said so.  Under a norm, whose weight may be an infinity or NaN,
        // what this token's q and k come to is left unwritten; else they are zeros
        // that are not turned.
        if (!known) {
          pos[0] = pos[1] = pos[2] = 0;
          if (c == 0 && f.h0 == 0) atomicExch(err, (int)CAST_ERR_INVALID_ARGUMENT);
          if constexpr (kNorm) {
            f.zeros(p.t[0], dst[0] + l * p.t[0].ds[1], p.t[0].ds[2]);
            if (!p.slots) f.zeros(p.t[1], dst[1] + l * p.t[1].ds[1], p.t[1].ds[2]);
            f.live = false;
          } else {
            f.blank = true;
            f.clear(raw);
#pragma unroll
            for (int j = 0; j < kC; ++j) f.turns[j] = false;
          }
        }
      }
      if (any_turns) {
        constexpr int kPieces = kHalf ? 1 : kC, kEach = kHalf ? 8 : 4;  // runs of pairs
#pragma unroll
        for (int j = 0; j < kPieces; ++j) {
          const int first = pair0 + j * (f.second >> 1);
          if (kPieces > 1 && !f.turns[j]) continue;
          const float2 *tab = reinterpret_cast<const float2 *>(p.table) + first;
          if (p.n_axes == 1) {
            const float4 *row = reinterpret_cast<const float4 *>(tab + pos[0] * half_pairs);
#pragma unroll
            for (int i = 0; i < kEach / 2; ++i) {
              const float4 w = __ldg(row + i);
              f.cs[kEach * j + 2 * i] = w.x, f.sn[kEach * j + 2 * i] = w.y;
              f.cs[kEach * j + 2 * i + 1] = w.z, f.sn[kEach * j + 2 * i + 1] = w.w;
            }
          } else {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
              const int r = first + i < p.axis_end0 ? pos[0] : first + i < p.axis_end1 ? pos[1] : pos[2];
              const float2 w = __ldg(tab + r * half_pairs + i);
              f.cs[kEach * j + i] = w.x, f.sn[kEach * j + i] = w.y;
            }
          }
        }
        // (kHalf: the second value of a pair takes y_b = z_b c + z_a s, the first y_a = z_a c - z_b s)
        if (flip) {
#pragma unroll
          for (int i = 0; i < kPairs; ++i) f.sn[i] = -f.sn[i];
        }
      }
    }
    f.template run<true>(p, p.t[0], src[0] + l * p.t[0].ss[1], dst[0] + l * p.t[0].ds[1], p.t[0].ds[2], raw);
    if (p.t[1].heads == 0) continue;  // uniform

    f.template load<!kNorm>(p, p.t[1], src[1] + l * p.t[1].ss[1], 0, raw);
    if (!p.slots) {
      f.template run<true>(p, p.t[1], src[1] + l * p.t[1].ss[1], dst[1] + l * p.t[1].ds[1], p.t[1].ds[2], raw);
      continue;
    }
    // place of this token's key and value in the cache
    long long place = -1;
    if (live_token) {
      const long long slot = load_index(p.slots, p.slots64, (long long)b * p.L + l);
      if (slot >= p.n_slots) {
        if (c == 0 && f.h0 == 0) atomicExch(err, (int)CAST_ERR_INVALID_ARGUMENT);
      } else if (slot >= 0) {
        const long long pg = slot <= 0x7fffffff ? (long long)((uint32_t)slot / (uint32_t)p.page) : slot / p.page;
        place = (pg * p.t[1].heads * p.page + (slot - pg * p.page)) * p.D;
      }
    }
    const long long head = (long long)p.page * p.D;
    const bool column = live_token && 8 * kC * c < p.D;
    if (kNorm && column && !f.live) {
      f.live = true;
      if (place >= 0) f.zeros(p.t[1], dst[1] + place, head);
      f.live = false;
    }
    f.template run<true>(p, p.t[1], src[1] + l * p.t[1].ss[1], place < 0 ? nullptr : dst[1] + place, head, raw);
    if (kNorm) f.live = column;  // (the value is copied whatever the position)
    f.template load<false>(p, p.t[2], src[2] + l * p.t[2].ss[1], 0, raw);
    f.template run<false>(p, p.t[2], src[2] + l * p.t[2].ss[1], place < 0 ? nullptr : dst[2] + place, head, raw);
  }
}

}  // namespace castk
