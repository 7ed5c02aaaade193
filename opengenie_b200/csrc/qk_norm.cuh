// Q/K RMSNorm and rotation in one pass, and its gradients.  For the columns x of one head (or of all heads of a
// row), r = rsqrt(mean(x^2) + eps):
//   y = R(x r w);   g = R^T(dy),  dw = sum over rows of g x r,  dx = r (g w) - x r^3 mean(g w x),
// where R turns the first `rotary` columns of each head by the token's angles (pairs (j, j + rotary/2), or
// neighbours (2j, 2j+1)) and leaves the others.  fp32 throughout, one bf16 rounding of y and dx; dw stays fp32.
//
// Both directions move every byte once: a team of 8- or 16-lane groups takes a token, a group takes a head at a
// time (8 columns per lane, one 16-byte load), and all of a group's heads are loaded before the first is used.
// The partner columns of a rotation and a head's sums travel by shuffles; a norm over the whole row adds the
// groups' sums through shared memory.
#pragma once

#include "elementwise.cuh"

namespace ogx {
namespace qkn {

constexpr int kThreads = 256;
enum Norm { kNone = 0, kHead = 1, kRow = 2 };

struct Params {
  const __nv_bfloat16 *x[2];   // q, k (rows of heads * HD columns)
  const __nv_bfloat16 *dy[2];  // gradients of the outputs (backward)
  __nv_bfloat16* y[2];         // outputs, or the gradients of q and k
  int64_t x_stride_b[2], x_stride_t[2], dy_stride_b[2], dy_stride_t[2], y_stride_b[2], y_stride_t[2];
  const void* weight[2];       // [HD] (head), [heads * HD] (row)
  const void *cos, *sin;       // [.., rotary / 2], element strides below
  int64_t cs_stride_b, cs_stride_h, cs_stride_t;
  int heads[2];
  int rotary;
  int interleaved;
  int w_fp32, cs_fp32;         // else bf16
  int team;                    // groups per token, a power of two
  int64_t tokens;              // per batch
  int64_t rows;                // batch * tokens
  float eps;
  float* partials;             // backward: [gridDim.x * teams][weight columns of q and k]
};

// Columns of the weight gradient (q's, then k's).
template <int HD, int NORM>
__device__ __forceinline__ int weight_columns(const Params& p) {
  return NORM == kHead ? 2 * HD : (p.heads[0] + p.heads[1]) * HD;
}

// 8 (or 4) values from entry `at` of a table of bf16 or fp32.
__device__ __forceinline__ void load8_of(const void* table, int64_t at, int fp32, float (&f)[8]) {
  if (fp32)
    load8(static_cast<const float*>(table) + at, f);
  else
    load8(static_cast<const __nv_bfloat16*>(table) + at, f);
}
__device__ __forceinline__ void load4_of(const void* table, int64_t at, int fp32, float (&f)[4]) {
  if (fp32) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(table) + at);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(table) + at);
    f[0] = __uint_as_float(v.x << 16);
    f[1] = __uint_as_float(v.x & 0xFFFF0000u);
    f[2] = __uint_as_float(v.y << 16);
    f[3] = __uint_as_float(v.y & 0xFFFF0000u);
  }
}

// This lane's cos and sin: entry i belongs to column i (half layout), entry i / 2 to columns i, i + 1
// (interleaved).  Lanes past the rotated columns get cos = 1, sin = 0.
__device__ __forceinline__ void load_angles(const Params& p, int64_t at, int sub, float (&c)[8], float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
  }
  if (sub * 8 >= p.rotary) return;
  if (p.interleaved) {
    float c4[4], s4[4];
    load4_of(p.cos, at + sub * 4, p.cs_fp32, c4);
    load4_of(p.sin, at + sub * 4, p.cs_fp32, s4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[2 * i] = c[2 * i + 1] = c4[i];
      s[2 * i] = -s4[i];
      s[2 * i + 1] = s4[i];
    }
  } else {
    const int half = p.rotary / 16;  // lanes of the first half
    const bool second = sub >= half;
    const int64_t entry = at + (second ? sub - half : sub) * 8;
    load8_of(p.cos, entry, p.cs_fp32, c);
    load8_of(p.sin, entry, p.cs_fp32, s);
    if (!second) {
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] = -s[i];
    }
  }
}

// x cos + partner sin (the sign of the first member's sine is in s); `inverse` turns back.
template <int LANES>
__device__ __forceinline__ void rotate(const Params& p, int sub, const float (&c)[8], const float (&s)[8], float inverse,
                                       float (&x)[8]) {
  if (p.interleaved) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const float a = x[i], b = x[i + 1];
      x[i] = fmaf(a, c[i], b * s[i] * inverse);
      x[i + 1] = fmaf(b, c[i + 1], a * s[i + 1] * inverse);
    }
  } else {
    const int half = p.rotary / 16;
    const int partner = sub < half ? sub + half : (sub < 2 * half ? sub - half : sub);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float o = __shfl_sync(0xffffffffu, x[i], partner, LANES);
      x[i] = fmaf(x[i], c[i], o * s[i] * inverse);
    }
  }
}

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int HD, int STEPS, int NORM, bool BACKWARD>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(Params p) {
  constexpr int LANES = HD / 8;
  constexpr int GROUPS = kThreads / LANES;
  __shared__ __align__(16) float sums[GROUPS][4];  // row norm: each group's sums (q: x^2, g w x; k: x^2, g w x)
  pdl_trigger();
  pdl_wait();
  const int sub = threadIdx.x % LANES;
  const int group = threadIdx.x / LANES;
  const int member = group % p.team;  // of the token's team
  const int team = group / p.team;
  const int teams = GROUPS / p.team;
  const int all_heads = p.heads[0] + p.heads[1];
  constexpr int DW = NORM == kRow ? STEPS : 2;  // weight-gradient accumulators of this lane: per head slot, or q and k
  float dw[BACKWARD && NORM != kNone ? DW : 1][8] = {};
  float w_head[NORM == kHead ? 2 : 1][8];
  if constexpr (NORM == kHead) {
    load8_of(p.weight[0], sub * 8, p.w_fp32, w_head[0]);
    load8_of(p.weight[1], sub * 8, p.w_fp32, w_head[1]);
  }

  // Every thread runs every iteration: shuffles and barriers name all of them.
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * teams; row0 < p.rows;
       row0 += static_cast<int64_t>(gridDim.x) * teams) {
    const int64_t row = row0 + team;
    const bool row_ok = row < p.rows;
    const int64_t batch = row_ok ? row / p.tokens : 0;
    const int64_t token = row_ok ? row - batch * p.tokens : 0;
    uint4 xr[STEPS], dr[BACKWARD ? STEPS : 1];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int h = member + i * p.team;
      const int t = h >= p.heads[0];
      const int64_t col = static_cast<int64_t>(h - (t ? p.heads[0] : 0)) * HD + sub * 8;
      xr[i] = make_uint4(0, 0, 0, 0);
      if (BACKWARD) dr[BACKWARD ? i : 0] = make_uint4(0, 0, 0, 0);
      if (row_ok && h < all_heads) {
        if (!(BACKWARD && NORM == kNone))
          xr[i] = __ldcs(reinterpret_cast<const uint4*>(p.x[t] + batch * p.x_stride_b[t] + token * p.x_stride_t[t] + col));
        if (BACKWARD)
          dr[BACKWARD ? i : 0] =
              __ldcs(reinterpret_cast<const uint4*>(p.dy[t] + batch * p.dy_stride_b[t] + token * p.dy_stride_t[t] + col));
      }
    }
    const int64_t angles = batch * p.cs_stride_b + token * p.cs_stride_t;
    float c[8], s[8];
    if (p.cs_stride_h == 0) load_angles(p, angles, sub, c, s);

    // row norm: both sums of the whole row first (the gradient's needs the turned-back g)
    float inv[2], along[2];
    if constexpr (NORM == kRow) {
      float sq[2] = {0.f, 0.f}, dot[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int h = member + i * p.team;
        const int t = h >= p.heads[0];
        float x[8];
        unpack8(xr[i], x);
        float a = 0.f, b = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) a = fmaf(x[e], x[e], a);
        if constexpr (BACKWARD) {
          float g[8], w[8] = {};
          unpack8(dr[i], g);
          const int ht = h < all_heads ? h - (t ? p.heads[0] : 0) : 0;
          if (p.cs_stride_h != 0) load_angles(p, angles + ht * p.cs_stride_h, sub, c, s);
          rotate<LANES>(p, sub, c, s, -1.f, g);
          if (h < all_heads) load8_of(p.weight[t], static_cast<int64_t>(ht) * HD + sub * 8, p.w_fp32, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) b = fmaf(g[e] * w[e], x[e], b);
        }
        sq[0] += t ? 0.f : a;
        sq[1] += t ? a : 0.f;
        dot[0] += t ? 0.f : b;
        dot[1] += t ? b : 0.f;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        sq[t] = group_sum<LANES>(sq[t]);
        if (BACKWARD) dot[t] = group_sum<LANES>(dot[t]);
      }
      __syncthreads();  // the previous row's sums have been read
      if (sub == 0) {
        sums[group][0] = sq[0];
        sums[group][1] = sq[1];
        sums[group][2] = dot[0];
        sums[group][3] = dot[1];
      }
      __syncthreads();
      sq[0] = sq[1] = dot[0] = dot[1] = 0.f;
      for (int m = 0; m < p.team; ++m) {
        const float4 v = *reinterpret_cast<const float4*>(sums[team * p.team + m]);
        sq[0] += v.x;
        sq[1] += v.y;
        dot[0] += v.z;
        dot[1] += v.w;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float n = 1.f / static_cast<float>(p.heads[t] * HD);
        inv[t] = rsqrtf(sq[t] * n + p.eps);
        along[t] = dot[t] * n * inv[t] * inv[t] * inv[t];
      }
    }

#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int h = member + i * p.team;
      const int t = h >= p.heads[0];
      const bool ok = row_ok && h < all_heads;
      const int hc = h < all_heads ? h : 0;
      const int ht = hc - (hc >= p.heads[0] ? p.heads[0] : 0);
      if (p.cs_stride_h != 0)  // a table for each head (q and k have the same heads)
        load_angles(p, angles + ht * p.cs_stride_h, sub, c, s);
      float x[8], w[8];
      unpack8(xr[i], x);
      if constexpr (NORM == kHead) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = t ? w_head[1][e] : w_head[0][e];
      } else if constexpr (NORM == kRow) {
        load8_of(p.weight[hc >= p.heads[0]], static_cast<int64_t>(ht) * HD + sub * 8, p.w_fp32, w);
      }
      if constexpr (!BACKWARD) {
        if constexpr (NORM != kNone) {
          float r;
          if constexpr (NORM == kHead) {
            float a = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) a = fmaf(x[e], x[e], a);
            r = rsqrtf(group_sum<LANES>(a) * (1.f / HD) + p.eps);
          } else {
            r = t ? inv[1] : inv[0];
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e];
        }
        rotate<LANES>(p, sub, c, s, 1.f, x);
      } else {
        float g[8];
        unpack8(dr[i], g);
        rotate<LANES>(p, sub, c, s, -1.f, g);
        if constexpr (NORM == kNone) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = g[e];
        } else {
          float r, al;
          if constexpr (NORM == kHead) {
            float a = 0.f, b = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              a = fmaf(x[e], x[e], a);
              b = fmaf(g[e] * w[e], x[e], b);
            }
            r = rsqrtf(group_sum<LANES>(a) * (1.f / HD) + p.eps);
            al = group_sum<LANES>(b) * (1.f / HD) * r * r * r;
          } else {
            r = t ? inv[1] : inv[0];
            al = t ? along[1] : along[0];
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float d = ok ? g[e] * (x[e] * r) : 0.f;
            if constexpr (NORM == kRow) {
              dw[i][e] += d;
            } else {
              dw[0][e] += t ? 0.f : d;
              dw[DW - 1][e] += t ? d : 0.f;
            }
            x[e] = fmaf(r, g[e] * w[e], -x[e] * al);
          }
        }
      }
      if (ok) {
        const int64_t col = static_cast<int64_t>(ht) * HD + sub * 8;
        __stcs(reinterpret_cast<uint4*>(p.y[t] + batch * p.y_stride_b[t] + token * p.y_stride_t[t] + col), pack8(x));
      }
    }
  }

  if constexpr (BACKWARD && NORM != kNone) {
    // this CTA's share of the weight gradients, summed over the rows it took
    if constexpr (NORM == kRow) {
      float* dst = p.partials + (static_cast<int64_t>(blockIdx.x) * teams + team) * (all_heads * HD);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int h = member + i * p.team;
        if (h < all_heads) {
          float4* d4 = reinterpret_cast<float4*>(dst + h * HD + sub * 8);
          d4[0] = make_float4(dw[i][0], dw[i][1], dw[i][2], dw[i][3]);
          d4[1] = make_float4(dw[i][4], dw[i][5], dw[i][6], dw[i][7]);
        }
      }
    } else {
      __shared__ float part[GROUPS][2 * HD];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        part[group][sub * 8 + e] = dw[0][e];
        part[group][HD + sub * 8 + e] = dw[DW - 1][e];
      }
      __syncthreads();
      for (int col = threadIdx.x; col < 2 * HD; col += kThreads) {
        float v = 0.f;
#pragma unroll
        for (int m = 0; m < GROUPS; ++m) v += part[m][col];
        p.partials[static_cast<int64_t>(blockIdx.x) * (2 * HD) + col] = v;
      }
    }
  }
}

// Sums the partial weight gradients over their rows in a fixed order: 32 columns per CTA, 32 slices of rows.
__global__ void __launch_bounds__(1024) qk_norm_weight_sum_kernel(const float* __restrict__ partials, int rows, int cols,
                                                                  int q_cols, float* dq_weight, float* dk_weight) {
  __shared__ float part[32][33];
  pdl_trigger();
  pdl_wait();
  const int col = blockIdx.x * 32 + (threadIdx.x & 31);
  const int slice = threadIdx.x >> 5;
  float v = 0.f;
  if (col < cols) {
#pragma unroll 4
    for (int r = slice; r < rows; r += 32) v += partials[static_cast<int64_t>(r) * cols + col];
  }
  part[slice][threadIdx.x & 31] = v;
  __syncthreads();
  if (slice == 0 && col < cols) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += part[i][threadIdx.x];
    if (col < q_cols)
      dq_weight[col] = v;
    else
      dk_weight[col - q_cols] = v;
  }
}

}  // namespace qkn
}  // namespace ogx
