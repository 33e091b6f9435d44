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
// Bound: HBM.  Every value is read and written once, in 16-byte pieces of
// eight values (two for float32), one lane a piece, so a head is a group of
// 8, 16 or 32 lanes of one warp: its sum of squares is a shuffle reduction and
// the half layout's partner values are a shuffle away, with no shared memory.
// A lane keeps the same eight columns for every head of its token, so the
// table row is read once per token and lane and its (c, s) stay in registers;
// kRotaryBatch heads are loaded before the first is worked on.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "compact.cuh"

namespace castk {

constexpr int kRotaryThreads = 128;
constexpr int kRotaryBatch = 4;  // heads in flight per lane

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
  long long tokens;  // B * L
  int L, D, R;
  int heads, lanes, slots_per_token, tokens_per_cta;  // lanes of one head; head groups of a token in a CTA
  int inverse, weight_f32, weight_per_head;
  float eps;
};

// Eight consecutive values as loaded, and their float32 values.
template <typename T>
struct Eight {
  uint4 w;
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
  float4 a, b;
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

template <typename InT, typename OutT, bool kNorm, bool kHalf>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  constexpr int kPairs = kHalf ? 8 : 4;  // table entries of a lane's eight columns
  int *err = &g_cast_device_error;
  const int group = threadIdx.x / p.lanes, c = threadIdx.x % p.lanes;
  const long long token = (long long)blockIdx.x * p.tokens_per_cta + group / p.slots_per_token;
  const bool live_token = group < p.slots_per_token * p.tokens_per_cta && token < p.tokens;
  const int h0 = group % p.slots_per_token;
  const bool live = live_token && 8 * c < p.D;
  const int b = live_token ? (int)(token / p.L) : 0;
  const int l = live_token ? (int)(token - (long long)b * p.L) : 0;

  // ---- this lane's (cos, sin): none where its columns are not rotated
  float cs[kPairs], sn[kPairs];
  const bool turns = live && 8 * c < p.R;
  bool known = true;  // every position of this token is a row of the table
  if (p.R > 0 && live_token) {
    long long pos[3];
#pragma unroll
    for (int a = 0; a < 3; ++a) {
      if (a < p.n_axes) {
        pos[a] = p.positions ? load_index(p.positions, p.pos64, b * p.pos_batch_stride + (long long)l * p.n_axes + a)
                             : p.first_position + l;
        if (pos[a] < 0 || pos[a] >= p.table_rows) {
          known = false;
          pos[a] = 0;
        }
      } else {
        pos[a] = pos[0];
      }
    }
    if (!known && c == 0 && h0 == 0) atomicExch(err, (int)CAST_ERR_INVALID_ARGUMENT);
    if (turns) {
      const int half_pairs = p.R / 2;
      const int p0 = kHalf ? (8 * c) % half_pairs : 4 * c;
      const float2 *tab = reinterpret_cast<const float2 *>(p.table);
      if (p.n_axes == 1) {
        const float4 *row = reinterpret_cast<const float4 *>(tab + pos[0] * half_pairs + p0);
#pragma unroll
        for (int i = 0; i < kPairs / 2; ++i) {
          const float4 w = __ldg(row + i);
          cs[2 * i] = w.x, sn[2 * i] = w.y, cs[2 * i + 1] = w.z, sn[2 * i + 1] = w.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) {
          const int pr = p0 + i;
          const long long r = pr < p.axis_end0 ? pos[0] : (pr < p.axis_end1 ? pos[1] : pos[2]);
          const float2 w = __ldg(tab + r * half_pairs + pr);
          cs[i] = w.x, sn[i] = w.y;
        }
      }
      // (kHalf: the second value of a pair reads y_b = z_b c + z_a s, the first y_a = z_a c - z_b s)
      const bool flip = (p.inverse != 0) != (kHalf && 8 * c < half_pairs);
      if (flip) {
#pragma unroll
        for (int i = 0; i < kPairs; ++i) sn[i] = -sn[i];
      }
    }
  }
  const int half_chunks = p.R / 16;
  const int partner = kHalf ? (threadIdx.x & 31) - c + (c < half_chunks ? c + half_chunks : c - half_chunks) : 0;

  long long slot = -1;
  if (p.slots && live_token) {
    slot = load_index(p.slots, p.slots64, token);
    if (slot >= p.n_slots) {
      if (c == 0 && h0 == 0) atomicExch(err, (int)CAST_ERR_INVALID_ARGUMENT);
      slot = -1;
    }
  }

  const int e1 = p.t[0].heads, e2 = e1 + p.t[1].heads;
  for (int hb = 0; hb < p.heads; hb += p.slots_per_token * kRotaryBatch) {  // same trip count in the whole CTA
    Eight<InT> raw[kRotaryBatch];
#pragma unroll
    for (int u = 0; u < kRotaryBatch; ++u) {
      const int h = hb + u * p.slots_per_token + h0;
      if (live && h < p.heads) {
        const int ti = h < e1 ? 0 : (h < e2 ? 1 : 2);
        const int th = h - (ti == 0 ? 0 : (ti == 1 ? e1 : e2));
        const RotaryTensor &t = p.t[ti];
        raw[u].load(static_cast<const InT *>(t.src) + b * t.ss[0] + l * t.ss[1] + th * t.ss[2] + 8 * c);
      }
    }
#pragma unroll
    for (int u = 0; u < kRotaryBatch; ++u) {
      const int h = hb + u * p.slots_per_token + h0;
      if (hb + u * p.slots_per_token >= p.heads) break;  // uniform
      const bool on = live && h < p.heads;
      const int ti = h < e1 ? 0 : (h < e2 ? 1 : 2);
      const int th = h - (ti == 0 ? 0 : (ti == 1 ? e1 : e2));
      const RotaryTensor &t = p.t[ti];
      float x[8];
      if (on) {
        raw[u].values(x);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.0f;
      }
      if (kNorm) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(x[i], x[i], sum);
        for (int s = p.lanes >> 1; s >= 1; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        if (on && t.weight) {
          const float r = rsqrtf(sum / (float)p.D + p.eps);
          const long long wo = (p.weight_per_head ? (long long)th * p.D : 0) + 8 * c;
          float w[8];
          if (p.weight_f32) {
            Eight<float> e;
            e.load(static_cast<const float *>(t.weight) + wo);
            e.values(w);
          } else {
            Eight<InT> e;
            e.load(static_cast<const InT *>(t.weight) + wo);
            e.values(w);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
        }
      }
      const bool rot = turns && ti < 2;
      if (kHalf) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float o = __shfl_sync(0xffffffffu, x[i], partner & 31);
          if (rot) x[i] = fmaf(x[i], cs[i], o * sn[i]);
        }
      } else if (rot) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float a = x[2 * i], q = x[2 * i + 1];
          x[2 * i] = fmaf(a, cs[i], -(q * sn[i]));
          x[2 * i + 1] = fmaf(a, sn[i], q * cs[i]);
        }
      }
      if (!on) continue;
      if (!known && ti < 2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.0f;
      }
      long long at;
      if (p.slots && ti > 0) {
        if (slot < 0) continue;
        const long long pg = slot / p.page;
        at = ((pg * t.heads + th) * p.page + (slot - pg * p.page)) * p.D;
      } else {
        at = b * t.ds[0] + l * t.ds[1] + th * t.ds[2];
      }
      store8(static_cast<OutT *>(t.dst) + at + 8 * c, x);
    }
  }
}

}  // namespace castk
