// Q/K RMSNorm and rotation in one pass, and its gradients.  For the columns x of one head (or of all heads of a
// row), r = rsqrt(mean(x^2) + eps):
//   y = R(x r w);   g = R^T(dy),  dw = sum over rows of g x r,  dx = r (g w) - x r^3 mean(g w x),
// where R turns the first `rotary` columns of each head by the token's angles (pairs (j, j + rotary/2), or
// neighbours (2j, 2j+1)) and leaves the others.  fp32 throughout, one bf16 rounding of y and dx; dw stays fp32.
//
// Both directions move every byte once.  HD / 8 lanes (a group) take a head, 8 columns each, and a team of groups
// takes a token.  A lane's columns are four first members of rotation pairs (`lo`) and their four partners
// (`hi`), so a rotation needs no other lane: two 8-byte loads at 4l and rotary/2 + 4l in the half layout; in the
// interleaved one the low and the high halves of four packed words.  Past the rotated columns a lane holds 8
// neighbours, with cos 1 and sin 0.  A head's sums travel by shuffles; a norm over the whole row adds the
// groups' sums through shared memory.  CTAs are persistent, and while one works on its tokens the next ones are
// on their way from HBM to L2 (bulk prefetches, which hold no registers).
#pragma once

#include "elementwise.cuh"

namespace ogx {
namespace qkn {

constexpr int kThreads = 256;
constexpr int kRowThreads = 512;  // a row norm keeps all of a token's columns in registers
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
  int w_fp32, cs_fp32;         // else bf16
  int team;                    // groups per token, a power of two
  int64_t tokens;              // per batch
  int64_t rows;                // batch * tokens
  float eps;
  float* partials;             // backward: [gridDim.x, or row norm gridDim.x * teams][weight columns of q and k]
};

// The 8 columns of a lane as 2 + 2 packed pairs.
struct Lane {
  f2 lo[2], hi[2];
};

template <bool INTER>
__device__ __forceinline__ Lane unpack_lane(const uint4& v) {
  Lane r;
  if constexpr (INTER) {
    r.lo[0] = f2{__uint_as_float(v.x << 16), __uint_as_float(v.y << 16)};
    r.lo[1] = f2{__uint_as_float(v.z << 16), __uint_as_float(v.w << 16)};
    r.hi[0] = f2{__uint_as_float(v.x & 0xFFFF0000u), __uint_as_float(v.y & 0xFFFF0000u)};
    r.hi[1] = f2{__uint_as_float(v.z & 0xFFFF0000u), __uint_as_float(v.w & 0xFFFF0000u)};
  } else {
    r.lo[0] = f2{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u)};
    r.lo[1] = f2{__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u)};
    r.hi[0] = f2{__uint_as_float(v.z << 16), __uint_as_float(v.z & 0xFFFF0000u)};
    r.hi[1] = f2{__uint_as_float(v.w << 16), __uint_as_float(v.w & 0xFFFF0000u)};
  }
  return r;
}

template <bool INTER>
__device__ __forceinline__ uint4 pack_lane(const Lane& r) {
  if constexpr (INTER)
    return make_uint4(pack_bf16x2(r.lo[0].x, r.hi[0].x), pack_bf16x2(r.lo[0].y, r.hi[0].y),
                      pack_bf16x2(r.lo[1].x, r.hi[1].x), pack_bf16x2(r.lo[1].y, r.hi[1].y));
  return make_uint4(pack_bf16x2(r.lo[0].x, r.lo[0].y), pack_bf16x2(r.lo[1].x, r.lo[1].y),
                    pack_bf16x2(r.hi[0].x, r.hi[0].y), pack_bf16x2(r.hi[1].x, r.hi[1].y));
}

// A lane's columns in memory: two runs of four, `hi` columns after `lo`'s start.
template <bool INTER>
struct Columns {
  int lo, gap;
  __device__ __forceinline__ Columns(const Params& p, int sub) {
    const int lanes = p.rotary / 8;  // that hold rotated columns
    if (INTER || sub >= lanes) {
      lo = sub * 8;
      gap = 4;
    } else {
      lo = sub * 4;
      gap = p.rotary / 2;
    }
  }
  __device__ __forceinline__ uint4 load(const __nv_bfloat16* head) const {
    if constexpr (INTER) return __ldcs(reinterpret_cast<const uint4*>(head + lo));
    const uint2 a = __ldcs(reinterpret_cast<const uint2*>(head + lo));
    const uint2 b = __ldcs(reinterpret_cast<const uint2*>(head + lo + gap));
    return make_uint4(a.x, a.y, b.x, b.y);
  }
  __device__ __forceinline__ void store(__nv_bfloat16* head, const uint4& v) const {
    if constexpr (INTER) {
      __stcs(reinterpret_cast<uint4*>(head + lo), v);
    } else {
      __stcs(reinterpret_cast<uint2*>(head + lo), make_uint2(v.x, v.y));
      __stcs(reinterpret_cast<uint2*>(head + lo + gap), make_uint2(v.z, v.w));
    }
  }
  // column of element e of (lo, hi) in the order of `Lane`: lo[0].x, lo[0].y, lo[1].x, .., hi[1].y
  __device__ __forceinline__ int column(int e) const {
    return INTER ? lo + 2 * (e & 3) + (e >> 2) : lo + (e & 3) + (e >> 2) * gap;
  }
};

__device__ __forceinline__ void load4_of(const void* table, int64_t at, int fp32, f2 (&f)[2]) {
  if (fp32) {
    const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(table) + at);
    f[0] = f2{v.x, v.y};
    f[1] = f2{v.z, v.w};
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(table) + at);
    f[0] = f2{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u)};
    f[1] = f2{__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u)};
  }
}

// cos and sin of a lane's four pairs; lanes past the rotated columns turn by nothing.  `sign` -1 turns back.
struct Angles {
  f2 c[2], s[2];
  __device__ __forceinline__ void load(const Params& p, int64_t at, int sub, float sign) {
    if (sub * 8 < p.rotary) {
      load4_of(p.cos, at + sub * 4, p.cs_fp32, c);
      load4_of(p.sin, at + sub * 4, p.cs_fp32, s);
    } else {
      c[0] = c[1] = f2{1.f, 1.f};
      s[0] = s[1] = f2{0.f, 0.f};
    }
    s[0] = mul2(s[0], f2{sign, sign});
    s[1] = mul2(s[1], f2{sign, sign});
  }
  __device__ __forceinline__ void turn(Lane& v) const {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f2 a = v.lo[i], b = v.hi[i];
      const f2 t = mul2(b, s[i]);
      v.lo[i] = fma2(a, c[i], f2{-t.x, -t.y});
      v.hi[i] = fma2(b, c[i], mul2(a, s[i]));
    }
  }
};

template <bool INTER>
__device__ __forceinline__ Lane load_weights(const Params& p, int t, int64_t at, const Columns<INTER>& col) {
  Lane w;
  if constexpr (INTER) {
    f2 a[2], b[2];
    load4_of(p.weight[t], at + col.lo, p.w_fp32, a);
    load4_of(p.weight[t], at + col.lo + 4, p.w_fp32, b);
    w.lo[0] = f2{a[0].x, a[1].x};
    w.lo[1] = f2{b[0].x, b[1].x};
    w.hi[0] = f2{a[0].y, a[1].y};
    w.hi[1] = f2{b[0].y, b[1].y};
  } else {
    load4_of(p.weight[t], at + col.lo, p.w_fp32, w.lo);
    load4_of(p.weight[t], at + col.lo + col.gap, p.w_fp32, w.hi);
  }
  return w;
}

__device__ __forceinline__ Lane mul(const Lane& a, const Lane& b) {
  return Lane{{mul2(a.lo[0], b.lo[0]), mul2(a.lo[1], b.lo[1])}, {mul2(a.hi[0], b.hi[0]), mul2(a.hi[1], b.hi[1])}};
}
__device__ __forceinline__ Lane mul(const Lane& a, float b) {
  const f2 v{b, b};
  return Lane{{mul2(a.lo[0], v), mul2(a.lo[1], v)}, {mul2(a.hi[0], v), mul2(a.hi[1], v)}};
}
// a * b + c
__device__ __forceinline__ Lane fma(const Lane& a, float b, const Lane& c) {
  const f2 v{b, b};
  return Lane{{fma2(a.lo[0], v, c.lo[0]), fma2(a.lo[1], v, c.lo[1])}, {fma2(a.hi[0], v, c.hi[0]), fma2(a.hi[1], v, c.hi[1])}};
}
__device__ __forceinline__ float dot(const Lane& a, const Lane& b) {
  f2 s = mul2(a.lo[0], b.lo[0]), t = mul2(a.hi[0], b.hi[0]);
  s = fma2(a.lo[1], b.lo[1], s);
  t = fma2(a.hi[1], b.hi[1], t);
  s = add2(s, t);
  return s.x + s.y;
}

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Brings `bytes` (a multiple of 16) of a later row to L2.
__device__ __forceinline__ void prefetch_row(const void* p, int bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// Prefetches row `row` of q, k and (backward) of their output gradients, one tensor per calling thread 0..3.
template <int HD, bool X, bool DY>
__device__ __forceinline__ void prefetch_token(const Params& p, int64_t row, int which) {
  const int t = which & 1;
  if (row >= p.rows) return;
  const int64_t batch = row / p.tokens, token = row - batch * p.tokens;
  if (which < 2 ? X : false) prefetch_row(p.x[t] + batch * p.x_stride_b[t] + token * p.x_stride_t[t], p.heads[t] * HD * 2);
  if (which >= 2 ? DY : false)
    prefetch_row(p.dy[t] + batch * p.dy_stride_b[t] + token * p.dy_stride_t[t], p.heads[t] * HD * 2);
}

// ------------------------------------------------------------------------- norm of each head, or no norm
// A group's heads are independent; UNROLL of them are loaded before the first is used.
template <int HD, int NORM, bool INTER, bool BACKWARD>
__global__ void __launch_bounds__(kThreads, BACKWARD ? 3 : 4) qk_head_kernel(Params p) {
  constexpr int LANES = HD / 8;
  constexpr int GROUPS = kThreads / LANES;
  constexpr int UNROLL = BACKWARD ? 2 : 4;
  constexpr bool X = NORM != kNone || !BACKWARD;
  __shared__ __align__(16) float weights[NORM == kHead ? 2 : 1][NORM == kHead ? HD : 4];  // lane by lane
  pdl_trigger();
  pdl_wait();
  const int sub = threadIdx.x % LANES;
  const int group = threadIdx.x / LANES;
  const int member = group % p.team;
  const int team = group / p.team;
  const int teams = GROUPS / p.team;
  const Columns<INTER> col(p, sub);
  if constexpr (NORM == kHead) {
    if (group < 2) {
      const Lane w = load_weights<INTER>(p, group, 0, col);
      *reinterpret_cast<Lane*>(&weights[group][sub * 8]) = w;
    }
    __syncthreads();
  }
  Lane dw[BACKWARD && NORM == kHead ? 2 : 1] = {};

  const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
  // whole warps run every iteration: the shuffles name all lanes
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * teams; row0 < p.rows; row0 += step) {
    if (threadIdx.x < 4 * teams) prefetch_token<HD, X, BACKWARD>(p, row0 + step + threadIdx.x / 4, threadIdx.x & 3);
    const int64_t row = row0 + team;
    const bool row_ok = row < p.rows;
    const int64_t batch = row_ok ? row / p.tokens : 0;
    const int64_t token = row_ok ? row - batch * p.tokens : 0;
    const int64_t angles = batch * p.cs_stride_b + token * p.cs_stride_t;
    Angles a;
    if (p.cs_stride_h == 0) a.load(p, angles, sub, BACKWARD ? -1.f : 1.f);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const __nv_bfloat16* xrow = p.x[t] + batch * p.x_stride_b[t] + token * p.x_stride_t[t];
      const __nv_bfloat16* drow = BACKWARD ? p.dy[t] + batch * p.dy_stride_b[t] + token * p.dy_stride_t[t] : nullptr;
      __nv_bfloat16* yrow = p.y[t] + batch * p.y_stride_b[t] + token * p.y_stride_t[t];
      for (int i0 = 0; i0 < p.heads[t]; i0 += UNROLL * p.team) {
        uint4 xr[UNROLL], dr[BACKWARD ? UNROLL : 1];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          const int h = i0 + u * p.team + member;
          const bool ok = row_ok && h < p.heads[t];
          if (X) xr[u] = ok ? col.load(xrow + h * HD) : make_uint4(0, 0, 0, 0);
          if constexpr (BACKWARD) dr[u] = ok ? col.load(drow + h * HD) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
          if (i0 + u * p.team >= p.heads[t]) break;  // the same for the whole CTA
          const int h = i0 + u * p.team + member;
          const bool ok = row_ok && h < p.heads[t];
          if (p.cs_stride_h != 0) a.load(p, angles + (ok ? h : 0) * p.cs_stride_h, sub, BACKWARD ? -1.f : 1.f);
          Lane v;
          if constexpr (!BACKWARD) {
            v = unpack_lane<INTER>(xr[u]);
            if constexpr (NORM == kHead) {
              const float r = rsqrtf(group_sum<LANES>(dot(v, v)) * (1.f / HD) + p.eps);
              v = mul(mul(v, r), *reinterpret_cast<const Lane*>(&weights[t][sub * 8]));
            }
            a.turn(v);
          } else {
            v = unpack_lane<INTER>(dr[u]);
            a.turn(v);
            if constexpr (NORM == kHead) {
              const Lane x = unpack_lane<INTER>(xr[u]);
              const Lane gw = mul(v, *reinterpret_cast<const Lane*>(&weights[t][sub * 8]));
              const float sq = group_sum<LANES>(dot(x, x)), gwx = group_sum<LANES>(dot(gw, x));
              const float r = rsqrtf(sq * (1.f / HD) + p.eps);
              const float along = gwx * (1.f / HD) * r * r * r;
              dw[t] = fma(mul(v, x), ok ? r : 0.f, dw[t]);  // idle slots hold zeros, whose r may be infinite
              v = fma(x, -along, mul(gw, r));
            }
          }
          if (ok) col.store(yrow + h * HD, pack_lane<INTER>(v));
        }
      }
    }
  }

  if constexpr (BACKWARD && NORM == kHead) {
    // this CTA's share of the weight gradients, summed over the rows it took
    __shared__ float part[GROUPS][2 * HD];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const float e[8] = {dw[t].lo[0].x, dw[t].lo[0].y, dw[t].lo[1].x, dw[t].lo[1].y,
                          dw[t].hi[0].x, dw[t].hi[0].y, dw[t].hi[1].x, dw[t].hi[1].y};
#pragma unroll
      for (int i = 0; i < 8; ++i) part[group][t * HD + col.column(i)] = e[i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * HD; c += kThreads) {
      float v = 0.f;
#pragma unroll
      for (int m = 0; m < GROUPS; ++m) v += part[m][c];
      p.partials[static_cast<int64_t>(blockIdx.x) * (2 * HD) + c] = v;
    }
  }
}

// ------------------------------------------------------------------------- norm over all heads of a row
// A team holds its token's columns (STEPS heads of q and of k per group) until the row's sums are known.
template <int HD, int STEPS, bool INTER, bool BACKWARD>
__global__ void __launch_bounds__(kRowThreads, STEPS == 1 ? 2 : 1) qk_row_kernel(Params p) {
  constexpr int LANES = HD / 8;
  constexpr int GROUPS = kRowThreads / LANES;
  __shared__ __align__(16) float sums[2][GROUPS][4];  // alternating rows: each group's q (x^2, g w x), k (x^2, g w x)
  pdl_trigger();
  pdl_wait();
  const int sub = threadIdx.x % LANES;
  const int group = threadIdx.x / LANES;
  const int member = group % p.team;
  const int team = group / p.team;
  const int teams = GROUPS / p.team;
  const Columns<INTER> col(p, sub);
  Lane dw[BACKWARD ? 2 : 1][BACKWARD ? STEPS : 1] = {};

  const int64_t step = static_cast<int64_t>(gridDim.x) * teams;
  int flip = 0;
  for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * teams; row0 < p.rows; row0 += step, flip ^= 1) {
    if (threadIdx.x < 4 * teams) prefetch_token<HD, true, BACKWARD>(p, row0 + step + threadIdx.x / 4, threadIdx.x & 3);
    const int64_t row = row0 + team;
    const bool row_ok = row < p.rows;
    const int64_t batch = row_ok ? row / p.tokens : 0;
    const int64_t token = row_ok ? row - batch * p.tokens : 0;
    const int64_t angles = batch * p.cs_stride_b + token * p.cs_stride_t;
    uint4 xr[2][STEPS], dr[BACKWARD ? 2 : 1][BACKWARD ? STEPS : 1];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int h = i * p.team + member;
        const bool ok = row_ok && h < p.heads[t];
        xr[t][i] = ok ? col.load(p.x[t] + batch * p.x_stride_b[t] + token * p.x_stride_t[t] + h * HD)
                      : make_uint4(0, 0, 0, 0);
        if constexpr (BACKWARD)
          dr[t][i] = ok ? col.load(p.dy[t] + batch * p.dy_stride_b[t] + token * p.dy_stride_t[t] + h * HD)
                        : make_uint4(0, 0, 0, 0);
      }
    }
    Angles a;
    if (p.cs_stride_h == 0) a.load(p, angles, sub, BACKWARD ? -1.f : 1.f);
    // the heads of q and k that a lane holds share their angles
    float part[2][2] = {};
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int h = i * p.team + member;
      if (BACKWARD && p.cs_stride_h != 0) a.load(p, angles + (h < p.heads[0] ? h : 0) * p.cs_stride_h, sub, -1.f);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const Lane x = unpack_lane<INTER>(xr[t][i]);
        part[t][0] += dot(x, x);
        if constexpr (BACKWARD) {
          Lane g = unpack_lane<INTER>(dr[t][i]);
          a.turn(g);
          const Lane w = load_weights<INTER>(p, t, static_cast<int64_t>(h < p.heads[t] ? h : 0) * HD, col);
          part[t][1] += dot(mul(g, w), x);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      part[t][0] = group_sum<LANES>(part[t][0]);
      if (BACKWARD) part[t][1] = group_sum<LANES>(part[t][1]);
    }
    if (sub == 0)
      *reinterpret_cast<float4*>(sums[flip][group]) = make_float4(part[0][0], part[0][1], part[1][0], part[1][1]);
    __syncthreads();  // the other half of `sums` is written only after every thread has passed here again
    float4 total = make_float4(0.f, 0.f, 0.f, 0.f);
    // lanes of a group take the team's sums in turn
    for (int m = sub; m < p.team; m += LANES) {
      const float4 v = *reinterpret_cast<const float4*>(sums[flip][team * p.team + m]);
      total.x += v.x;
      total.y += v.y;
      total.z += v.z;
      total.w += v.w;
    }
    const float sq[2] = {group_sum<LANES>(total.x), group_sum<LANES>(total.z)};
    float gwx[2] = {0.f, 0.f};
    if constexpr (BACKWARD) {
      gwx[0] = group_sum<LANES>(total.y);
      gwx[1] = group_sum<LANES>(total.w);
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int h = i * p.team + member;
      if (p.cs_stride_h != 0)
        a.load(p, angles + (h < p.heads[0] ? h : 0) * p.cs_stride_h, sub, BACKWARD ? -1.f : 1.f);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float n = 1.f / static_cast<float>(p.heads[t] * HD);
        const float r = rsqrtf(sq[t] * n + p.eps);
        const bool ok = row_ok && h < p.heads[t];
        const Lane w = load_weights<INTER>(p, t, static_cast<int64_t>(h < p.heads[t] ? h : 0) * HD, col);
        Lane v;
        if constexpr (!BACKWARD) {
          v = mul(mul(unpack_lane<INTER>(xr[t][i]), r), w);
          a.turn(v);
        } else {
          const Lane x = unpack_lane<INTER>(xr[t][i]);
          Lane g = unpack_lane<INTER>(dr[t][i]);
          a.turn(g);
          dw[t][i] = fma(mul(g, x), ok ? r : 0.f, dw[t][i]);
          v = fma(x, -(gwx[t] * n * r * r * r), mul(mul(g, w), r));
        }
        if (ok)
          col.store(p.y[t] + batch * p.y_stride_b[t] + token * p.y_stride_t[t] + h * HD, pack_lane<INTER>(v));
      }
    }
  }

  if constexpr (BACKWARD) {
    const int columns = (p.heads[0] + p.heads[1]) * HD;
    float* dst = p.partials + (static_cast<int64_t>(blockIdx.x) * teams + team) * columns;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int h = i * p.team + member;
        if (h < p.heads[t]) {
          const float e[8] = {dw[t][i].lo[0].x, dw[t][i].lo[0].y, dw[t][i].lo[1].x, dw[t][i].lo[1].y,
                              dw[t][i].hi[0].x, dw[t][i].hi[0].y, dw[t][i].hi[1].x, dw[t][i].hi[1].y};
#pragma unroll
          for (int k = 0; k < 8; ++k) dst[(t * p.heads[0] + h) * HD + col.column(k)] = e[k];
        }
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
#pragma unroll 8
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
