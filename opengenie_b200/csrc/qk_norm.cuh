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
// groups' sums through shared memory.  A CTA works on q or on k (CTAs shared out by the heads), is persistent,
// and while it works on its tokens the next ones are on their way from HBM to L2 (bulk prefetches by one warp,
// which hold no registers).  Integer work per token would cost more issue slots than the norm: a thread keeps one
// address per tensor and steps it by strides that the host has multiplied out.
#pragma once

#include "elementwise.cuh"

namespace ogx {
namespace qkn {

constexpr int kThreads = 256;
enum Norm { kNone = 0, kHead = 1, kRow = 2 };
// Resident CTAs per SM that the kernels are compiled for; a launch has at most one wave of them.
__host__ __device__ constexpr int head_ctas(bool backward) { return backward ? 3 : 4; }
__host__ __device__ constexpr int row_ctas(int threads, int steps) { return threads == 256 ? (steps == 1 ? 3 : 2) : 1; }

// Rows of a tensor: the address of (batch, token) and the steps from a team's token to its next one (`wrap` more
// when that crosses into another batch).  Bytes.
struct Stream {
  char* base;
  int64_t stride_b, stride_t;
  int64_t step, wrap;
};

// One of q and k.
struct Tensor {
  Stream x, dy, y;     // input rows; gradients of the output rows (backward); output rows or the input's gradients
  Stream angles;       // offsets into cos and sin (base null)
  const void* weight;  // [HD] (head), [heads * HD] (row)
  float* partials;     // backward: [CTAs (head) or CTAs * teams (row)][weight columns]
  int heads;
  int team;            // groups per token, a power of two
  int ctas;
  int step_token;      // tokens (of a batch) from a team's token to its next one, batches left out
};

struct Params {
  Tensor t[2];               // CTAs [0, t[0].ctas) take q, the rest k
  const char *cos, *sin;     // [.., rotary / 2]
  int64_t cs_stride_h;       // bytes; 0: shared by the heads
  int rotary;
  int w_fp32, cs_fp32;       // else bf16
  int tokens;                // per batch
  int rows;                  // batch * tokens
  float eps;
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
  // `at`: the address of the lane's first column
  __device__ __forceinline__ uint4 load(const char* at) const {
    if constexpr (INTER) return __ldcs(reinterpret_cast<const uint4*>(at));
    const uint2 a = __ldcs(reinterpret_cast<const uint2*>(at));
    const uint2 b = __ldcs(reinterpret_cast<const uint2*>(at + gap * 2));
    return make_uint4(a.x, a.y, b.x, b.y);
  }
  __device__ __forceinline__ void store(char* at, const uint4& v) const {
    if constexpr (INTER) {
      __stcs(reinterpret_cast<uint4*>(at), v);
    } else {
      __stcs(reinterpret_cast<uint2*>(at), make_uint2(v.x, v.y));
      __stcs(reinterpret_cast<uint2*>(at + gap * 2), make_uint2(v.z, v.w));
    }
  }
  // column of element e of (lo, hi) in the order of `Lane`: lo[0].x, lo[0].y, lo[1].x, .., hi[1].y
  __device__ __forceinline__ int column(int e) const {
    return INTER ? lo + 2 * (e & 3) + (e >> 2) : lo + (e & 3) + (e >> 2) * gap;
  }
};

// Four entries, from entry `entry` on, of the fp32 or bf16 values at `at`.
__device__ __forceinline__ void load4_of(const char* at, int entry, int fp32, f2 (&f)[2]) {
  if (fp32) {
    const float4 v = *reinterpret_cast<const float4*>(at + entry * 4);
    f[0] = f2{v.x, v.y};
    f[1] = f2{v.z, v.w};
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(at + entry * 2);
    f[0] = f2{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u)};
    f[1] = f2{__uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u)};
  }
}

// Where a lane finds its four pairs' angles: the address of its cos entries, and sin's distance from it.
struct AngleRow {
  const char* cos;
  int64_t to_sin;
  int fp32;
  bool turned;  // false: the lane's columns lie past the rotated ones
  __device__ __forceinline__ AngleRow(const Params& p, int64_t at, int sub)
      : cos(p.cos + at + sub * (p.cs_fp32 ? 16 : 8)), to_sin(p.sin - p.cos), fp32(p.cs_fp32), turned(sub * 8 < p.rotary) {}
};

// cos and sin of a lane's four pairs, for the rotation or (BACK) for turning back; columns that do not turn have 1, 0.
struct Turn {
  f2 c[2], s[2], ns[2];
  template <bool BACK>
  __device__ __forceinline__ void load(const AngleRow& a, int64_t offset) {
    f2 t[2];
    if (a.turned) {
      load4_of(a.cos + offset, 0, a.fp32, c);
      load4_of(a.cos + offset + a.to_sin, 0, a.fp32, t);
    } else {
      c[0] = c[1] = f2{1.f, 1.f};
      t[0] = t[1] = f2{0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f2 n = mul2(t[i], f2{-1.f, -1.f});
      s[i] = BACK ? n : t[i];
      ns[i] = BACK ? t[i] : n;
    }
  }
  __device__ __forceinline__ Lane operator()(const Lane& v) const {
    Lane r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      r.lo[i] = fma2(v.hi[i], ns[i], mul2(v.lo[i], c[i]));
      r.hi[i] = fma2(v.lo[i], s[i], mul2(v.hi[i], c[i]));
    }
    return r;
  }
};

// The weight and the rotation as one step: R(w o x).
struct WeightedTurn {
  f2 ll[2], lh[2], hl[2], hh[2];
  __device__ __forceinline__ WeightedTurn(const Turn& t, const Lane& w) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      ll[i] = mul2(t.c[i], w.lo[i]);
      lh[i] = mul2(t.ns[i], w.hi[i]);
      hl[i] = mul2(t.s[i], w.lo[i]);
      hh[i] = mul2(t.c[i], w.hi[i]);
    }
  }
  __device__ __forceinline__ Lane operator()(const Lane& v) const {
    Lane r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      r.lo[i] = fma2(v.hi[i], lh[i], mul2(v.lo[i], ll[i]));
      r.hi[i] = fma2(v.lo[i], hl[i], mul2(v.hi[i], hh[i]));
    }
    return r;
  }
};

template <bool INTER>
__device__ __forceinline__ Lane load_weights(const void* weights, int fp32, int at, const Columns<INTER>& col) {
  const char* weight = static_cast<const char*>(weights);
  Lane w;
  if constexpr (INTER) {
    f2 a[2], b[2];
    load4_of(weight, at + col.lo, fp32, a);
    load4_of(weight, at + col.lo + 4, fp32, b);
    w.lo[0] = f2{a[0].x, a[1].x};
    w.lo[1] = f2{b[0].x, b[1].x};
    w.hi[0] = f2{a[0].y, a[1].y};
    w.hi[1] = f2{b[0].y, b[1].y};
  } else {
    load4_of(weight, at + col.lo, fp32, w.lo);
    load4_of(weight, at + col.lo + col.gap, fp32, w.hi);
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

// A CTA's place: its tensor and which of the tensor's CTAs it is.
struct Place {
  int tensor, cta;
  __device__ __forceinline__ explicit Place(const Params& p) {
    tensor = static_cast<int>(blockIdx.x) >= p.t[0].ctas;
    cta = static_cast<int>(blockIdx.x) - (tensor ? p.t[0].ctas : 0);
  }
};

__device__ __forceinline__ char* row_address(const Stream& s, int batch, int token) {
  return s.base + batch * s.stride_b + token * s.stride_t;
}

// A team's token, stepping through the rows with additions.
struct Cursor {
  int row, token;
  bool wrapped;  // the last step crossed into another batch
  __device__ __forceinline__ void step(const Params& p, const Tensor& a, int rows) {
    row += rows;
    token += a.step_token;
    wrapped = token >= p.tokens;
    if (wrapped) token -= p.tokens;
  }
};
__device__ __forceinline__ int64_t step_of(const Stream& s, bool wrapped) { return wrapped ? s.step + s.wrap : s.step; }

// The rows of the CTA's tokens [row0, row0 + teams) to L2, by its first warp.
template <int HD, bool X, bool DY>
__device__ __forceinline__ void prefetch_rows(const Params& p, const Tensor& a, int row0, int teams) {
  if (threadIdx.x >= 32) return;
  for (int i = threadIdx.x; i < 2 * teams; i += 32) {
    const int row = row0 + (i >> 1);
    if (row >= p.rows) break;
    const int batch = row / p.tokens, token = row - batch * p.tokens;
    if (X && (i & 1) == 0) prefetch_row(row_address(a.x, batch, token), a.heads * HD * 2);
    if (DY && (i & 1) == 1) prefetch_row(row_address(a.dy, batch, token), a.heads * HD * 2);
  }
}

// Its part of a head's angles to L2, by each lane (bulk prefetches of so small pieces, one lane after the other,
// took longer than the rows themselves).
__device__ __forceinline__ void prefetch_angles(const AngleRow& a, int64_t offset) {
  if (!a.turned) return;
  asm volatile("prefetch.global.L2 [%0];" ::"l"(a.cos + offset));
  asm volatile("prefetch.global.L2 [%0];" ::"l"(a.cos + offset + a.to_sin));
}

__device__ __forceinline__ void elements(const Lane& v, float (&e)[8]) {
  e[0] = v.lo[0].x; e[1] = v.lo[0].y; e[2] = v.lo[1].x; e[3] = v.lo[1].y;
  e[4] = v.hi[0].x; e[5] = v.hi[0].y; e[6] = v.hi[1].x; e[7] = v.hi[1].y;
}

// ------------------------------------------------------------------------- norm of each head, or no norm
// A group's heads are independent; UNROLL of them are loaded before the first is used.  Bound by HBM: 9216 tokens of
// 32 + 32 heads 51 us = 6.0 TB/s (92 % of a plain copy), their gradient 82 us = 5.6 TB/s with its sums of the weights'
// gradients; 4 tokens 2 us.
template <int HD, int NORM, bool INTER, bool PER_HEAD, bool BACKWARD>
__global__ void __launch_bounds__(kThreads, head_ctas(BACKWARD)) qk_head_kernel(const __grid_constant__ Params p) {
  constexpr int LANES = HD / 8;
  constexpr int GROUPS = kThreads / LANES;
  constexpr int UNROLL = BACKWARD ? 2 : 4;
  constexpr bool X = NORM != kNone || !BACKWARD;
  pdl_trigger();
  pdl_wait();
  const Place place(p);
  const Tensor& a = p.t[place.tensor];
  const int sub = threadIdx.x % LANES;
  const int group = threadIdx.x / LANES;
  const int heads = a.heads, stride = a.team;
  const int member = group & (stride - 1);
  const int team = group / stride;
  const int teams = GROUPS / stride;
  const Columns<INTER> col(p, sub);
  Lane w;
  if constexpr (NORM == kHead) w = load_weights<INTER>(a.weight, p.w_fp32, 0, col);
  Lane dw{};

  const int rows_per_step = a.ctas * teams;
  Cursor at{place.cta * teams + team, 0, false};
  const int batch0 = at.row / p.tokens;
  at.token = at.row - batch0 * p.tokens;
  const int offset = (member * HD + col.lo) * 2;
  const char* xp = row_address(a.x, batch0, at.token) + offset;
  const char* dp = BACKWARD ? row_address(a.dy, batch0, at.token) + offset : nullptr;
  char* yp = row_address(a.y, batch0, at.token) + offset;
  AngleRow angles(p, batch0 * a.angles.stride_b + at.token * a.angles.stride_t + (PER_HEAD ? member * p.cs_stride_h : 0), sub);
  uint4 xr[UNROLL] = {}, dr[UNROLL] = {};  // idle slots keep what was there before, and write nothing
  // whole warps run every iteration: the shuffles name all lanes
  for (int row0 = place.cta * teams; row0 < p.rows; row0 += rows_per_step) {
    prefetch_rows<HD, X, BACKWARD>(p, a, row0 + rows_per_step, teams);
    const bool row_ok = at.row < p.rows;
    Turn turn{};
    if constexpr (!PER_HEAD) {
      if (row_ok) turn.load<BACKWARD>(angles, 0);
    }
    const WeightedTurn step1(turn, w);  // used by the forward pass of a norm with shared tables
    for (int i0 = 0; i0 < heads; i0 += UNROLL * stride) {
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int h = i0 + u * stride;
        if (row_ok && h + member < heads) {
          if constexpr (X) xr[u] = col.load(xp + h * (HD * 2));
          if constexpr (BACKWARD) dr[u] = col.load(dp + h * (HD * 2));
        }
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int h = i0 + u * stride;
        if (h >= heads) break;  // the same for the whole CTA
        const bool ok = row_ok && h + member < heads;
        if constexpr (PER_HEAD) {
          if (ok) turn.load<BACKWARD>(angles, h * p.cs_stride_h);
        }
        Lane v;
        if constexpr (NORM == kNone) {
          v = turn(unpack_lane<INTER>(BACKWARD ? dr[u] : xr[u]));
        } else if constexpr (!BACKWARD) {
          const Lane x = unpack_lane<INTER>(xr[u]);
          const float inv = rsqrtf(group_sum<LANES>(dot(x, x)) * (1.f / HD) + p.eps);
          v = mul(PER_HEAD ? turn(mul(x, w)) : step1(x), inv);
        } else {
          const Lane x = unpack_lane<INTER>(xr[u]);
          const Lane g = turn(unpack_lane<INTER>(dr[u]));
          const Lane gx = mul(g, x);
          const float sq = group_sum<LANES>(dot(x, x)), gwx = group_sum<LANES>(dot(gx, w));
          const float inv = rsqrtf(sq * (1.f / HD) + p.eps);
          if (ok) dw = fma(gx, inv, dw);
          v = fma(x, -gwx * (1.f / HD) * inv * inv * inv, mul(mul(g, w), inv));
        }
        if (ok) col.store(yp + h * (HD * 2), pack_lane<INTER>(v));
      }
    }
    at.step(p, a, rows_per_step);
    if constexpr (X) xp += step_of(a.x, at.wrapped);
    if constexpr (BACKWARD) dp += step_of(a.dy, at.wrapped);
    yp += step_of(a.y, at.wrapped);
    angles.cos += step_of(a.angles, at.wrapped);
  }

  if constexpr (BACKWARD && NORM == kHead) {
    // this CTA's share of the weight gradient, summed over the rows it took
    __shared__ float part[GROUPS][HD];
    float e[8];
    elements(dw, e);
#pragma unroll
    for (int i = 0; i < 8; ++i) part[group][col.column(i)] = e[i];
    __syncthreads();
    if (threadIdx.x < HD) {
      float v = 0.f;
#pragma unroll
      for (int m = 0; m < GROUPS; ++m) v += part[m][threadIdx.x];
      a.partials[static_cast<int64_t>(place.cta) * HD + threadIdx.x] = v;
    }
  }
}

// ------------------------------------------------------------------------- norm over all heads of a row
// A team holds its token's columns (STEPS heads per group) until the row's sums are known.  Bound by instructions and the
// wait for those sums (16 warps on an SM, a half of the issue slots used): 9216 tokens of 32 + 32 heads with tables for
// each head 111 us = 3.4 TB/s, the gradient 150 us = 3.5 TB/s.  More than 64 heads of 128 take four heads to a
// group, and their gradient spills registers (0.5 KB a thread): 4608 tokens with tables for all heads, 64 + 64 heads 98
// and 144 us, 96 + 32 heads, the same bytes, 208 and 445.
template <int HD, int THREADS, int STEPS, bool INTER, bool PER_HEAD, bool BACKWARD>
__global__ void __launch_bounds__(THREADS, row_ctas(THREADS, STEPS)) qk_row_kernel(const __grid_constant__ Params p) {
  constexpr int LANES = HD / 8;
  constexpr int GROUPS = THREADS / LANES;
  __shared__ __align__(8) float sums[2][GROUPS][2];  // alternating rows: each group's sums of x^2 and g w x
  pdl_trigger();
  pdl_wait();
  const Place place(p);
  const Tensor& a = p.t[place.tensor];
  const int sub = threadIdx.x % LANES;
  const int group = threadIdx.x / LANES;
  const int heads = a.heads, stride = a.team;
  const int member = group & (stride - 1);
  const int team = group / stride;
  const int teams = GROUPS / stride;
  const Columns<INTER> col(p, sub);
  const float n = 1.f / static_cast<float>(heads * HD);
  Lane dw[STEPS] = {};
  // the weights of the group's heads stay in registers (four heads would not fit: they are read again)
  constexpr bool KEEP = STEPS <= 2;
  Lane w[STEPS];
  const auto weights_of = [&](int i) {
    const int h = i * stride + member;
    return load_weights<INTER>(a.weight, p.w_fp32, (h < heads ? h : 0) * HD, col);
  };
  if constexpr (KEEP) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) w[i] = weights_of(i);
  }

  const int rows_per_step = a.ctas * teams;
  Cursor at{place.cta * teams + team, 0, false};
  const int batch0 = at.row / p.tokens;
  at.token = at.row - batch0 * p.tokens;
  const int offset = (member * HD + col.lo) * 2;
  const char* xp = row_address(a.x, batch0, at.token) + offset;
  const char* dp = BACKWARD ? row_address(a.dy, batch0, at.token) + offset : nullptr;
  char* yp = row_address(a.y, batch0, at.token) + offset;
  const int64_t head_step = stride * p.cs_stride_h;  // to the angles of the group's next head
  AngleRow angles(p, batch0 * a.angles.stride_b + at.token * a.angles.stride_t + (PER_HEAD ? member * p.cs_stride_h : 0), sub);
  // groups past the last head keep zeros; a team past the last row keeps its last one, and writes nothing
  uint4 xr[STEPS] = {}, dr[STEPS] = {};
  const auto load_row = [&](bool ok) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (ok && i * stride + member < heads) {
        xr[i] = col.load(xp + i * stride * (HD * 2));
        if constexpr (BACKWARD) dr[i] = col.load(dp + i * stride * (HD * 2));
      }
    }
  };
  load_row(at.row < p.rows);
  int flip = 0;
  for (int row0 = place.cta * teams; row0 < p.rows; row0 += rows_per_step, flip ^= 1) {
    prefetch_rows<HD, true, BACKWARD>(p, a, row0 + 2 * rows_per_step, teams);
    const bool row_ok = at.row < p.rows;
    at.step(p, a, rows_per_step);
    const int64_t to_next = step_of(a.angles, at.wrapped);
    if (PER_HEAD && at.row < p.rows) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
        if (i * stride + member < heads) prefetch_angles(angles, to_next + i * head_step);
    }
    Turn turn{};
    if (!PER_HEAD && row_ok) turn.load<BACKWARD>(angles, 0);
    Lane x[STEPS], g[STEPS];
    float sq = 0.f, gwx = 0.f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int h = i * stride + member;
      x[i] = unpack_lane<INTER>(xr[i]);
      sq += dot(x[i], x[i]);
      if ((BACKWARD || STEPS == 1) && PER_HEAD && row_ok && h < heads) turn.load<BACKWARD>(angles, i * head_step);
      if constexpr (BACKWARD) {
        if constexpr (!KEEP) w[i] = weights_of(i);
        g[i] = turn(unpack_lane<INTER>(dr[i]));
        gwx += dot(mul(g[i], w[i]), x[i]);
      }
    }
    // the next row's loads run behind this row's sums and outputs
    xp += step_of(a.x, at.wrapped);
    if constexpr (BACKWARD) dp += step_of(a.dy, at.wrapped);
    load_row(at.row < p.rows);
    sq = group_sum<LANES>(sq);
    if constexpr (BACKWARD) gwx = group_sum<LANES>(gwx);
    if (sub == 0) *reinterpret_cast<float2*>(sums[flip][group]) = make_float2(sq, gwx);
    __syncthreads();  // the other half of `sums` is written only after every thread has passed here again
    sq = gwx = 0.f;
    for (int m = sub; m < stride; m += LANES) {
      const float2 v = *reinterpret_cast<const float2*>(sums[flip][team * stride + m]);
      sq += v.x;
      gwx += v.y;
    }
    sq = group_sum<LANES>(sq);
    const float inv = rsqrtf(sq * n + p.eps);
    float along = 0.f;
    if constexpr (BACKWARD) along = -group_sum<LANES>(gwx) * n * inv * inv * inv;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int h = i * stride + member;
      const bool ok = row_ok && h < heads;
      Lane v;
      if constexpr (!BACKWARD) {
        // with one head per group its angles are still there
        if (STEPS > 1 && PER_HEAD && ok) turn.load<BACKWARD>(angles, i * head_step);
        if constexpr (!KEEP) w[i] = weights_of(i);
        v = turn(mul(mul(x[i], inv), w[i]));
      } else {
        if constexpr (!KEEP) w[i] = weights_of(i);
        if (ok) dw[i] = fma(mul(g[i], x[i]), inv, dw[i]);
        v = fma(x[i], along, mul(mul(g[i], w[i]), inv));
      }
      if (ok) col.store(yp + i * stride * (HD * 2), pack_lane<INTER>(v));
    }
    yp += step_of(a.y, at.wrapped);
    angles.cos += to_next;
  }

  if constexpr (BACKWARD) {
    float* dst = a.partials + (static_cast<int64_t>(place.cta) * teams + team) * (heads * HD);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int h = i * stride + member;
      if (h < heads) {
        float e[8];
        elements(dw[i], e);
#pragma unroll
        for (int k = 0; k < 8; ++k) dst[h * HD + col.column(k)] = e[k];
      }
    }
  }
}

// Sums the partial weight gradients of q (and behind them of k) over their rows in a fixed order: 32 columns per
// CTA, 32 slices of rows.
struct SumParams {
  const float* partials[2];
  float* out[2];
  int rows[2], cols[2];
};

__global__ void __launch_bounds__(1024) qk_norm_weight_sum_kernel(const __grid_constant__ SumParams p) {
  __shared__ float part[32][33];
  pdl_trigger();
  pdl_wait();
  const int q_ctas = (p.cols[0] + 31) / 32;
  const int t = static_cast<int>(blockIdx.x) >= q_ctas;
  const int cols = p.cols[t], rows = p.rows[t];
  const int col = (static_cast<int>(blockIdx.x) - (t ? q_ctas : 0)) * 32 + (threadIdx.x & 31);
  const int slice = threadIdx.x >> 5;
  float v = 0.f;
  if (col < cols) {
    const float* src = p.partials[t] + col;
#pragma unroll 16
    for (int r = slice; r < rows; r += 32) v += src[static_cast<int64_t>(r) * cols];
  }
  part[slice][threadIdx.x & 31] = v;
  __syncthreads();
  if (slice == 0 && col < cols) {
    v = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v += part[i][threadIdx.x];
    p.out[t][col] = v;
  }
}

}  // namespace qkn
}  // namespace ogx
