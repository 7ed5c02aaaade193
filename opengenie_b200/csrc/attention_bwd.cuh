// Gradients of attention, head_dim 128, bf16 in and out, fp32 softmax and accumulation.  With c the softmax
// scale, S = c Q K^T, P = exp(S - lse) (recomputed from the row statistics the forward pass kept) and
// delta_i = dO_i . O_i:
//   dV = P^T dO,   dP = dO V^T,   dS = P o (dP - delta),   dQ = c dS K,   dK = c dS^T Q;
// dK and dV of a shared key/value head sum over its query heads.
//
// attn_bwd_stats_kernel writes per query row -lse * log2(e) and -delta.  attn_bwd_kernel has a CTA for every tile
// of 128 keys of a key/value head (dK and dV, over all query tiles of its query heads) and a CTA for every tile of
// 128 queries of a head (dQ, over all key tiles).  S and dP are computed in both: seven tile products instead of
// five.  In return every gradient is summed in one CTA's tensor memory in a fixed order: no fp32 buffer for dQ, no
// atomics, and the same bits on every run.  (The five-product form adds its dQ tiles to HBM, a 64 KB reduction per
// tile pair, in whatever order the CTAs reach it unless each waits for its turn.)  Where one side has so few tiles that
// the GPU would idle behind long sums, several CTAs share a sum and attn_bwd_join_kernel adds their parts, in their order.
//
// What bounds it, at 9216 x 9216 x 32 heads: 3.71 ms back to back, under the 1000 W cap (1.43 GHz) 1312 TFLOP/s of
// its seven products, 96 % of what cuBLAS sustains there; 3.20 ms in a burst.  Per tile pair the two roles take 2700
// and 1900 cycles for 2048 and 1536 of products: the S and dP products use the whole 128 bytes per clock of shared
// memory, so that every TMA write (64 KB a pair) delays them, and a CTA spends about 9000 cycles on starting (TMA
// latency, first scores) and storing.
//
// P and dS are rounded to bf16, the type that the instruction wants where the other operand is bf16: each term of a sum
// by 2^-8 at most, which leaves the gradients 0.0023 to 0.0024 of their norm from the exact ones where their own rounding
// leaves 0.0017.  The degree-3 polynomial's 7.5e-5 disappears beside it.
#pragma once

#include "attention_masked.cuh"
#include "rows.cuh"

namespace ogx {
namespace attn {

constexpr int BT = 128;                        // queries or keys per tile
constexpr int T_HALF_BYTES = BT * 64 * 2;      // 64-column half of a tile (128-byte rows, 128-byte swizzle)
constexpr int T_BYTES = 2 * T_HALF_BYTES;
constexpr int STAT_FLOATS = 2 * BT;            // a query tile's statistics: 128 x -lse*log2e, 128 x -delta
constexpr int STAT_BYTES = STAT_FLOATS * 4;
constexpr int B_STAGES = 2;                    // ring of the operands a CTA streams
constexpr int DQ_K_STAGES = 3;                 // K tiles of a dQ CTA: S of the next tile but one needs its K early
constexpr int BWD_SMEM_DKDV = (2 + 2 * B_STAGES) * T_BYTES + B_STAGES * STAT_BYTES;
constexpr int BWD_SMEM_DQ = (2 + B_STAGES + DQ_K_STAGES) * T_BYTES;
constexpr int BWD_SMEM = (BWD_SMEM_DKDV > BWD_SMEM_DQ ? BWD_SMEM_DKDV : BWD_SMEM_DQ) + 1024;
constexpr int kBwdThreads = 384;               // TMA, MMA, row-zeroing and one idle warp; two softmax groups
constexpr int kSoftmaxWarps = 8;
constexpr int kAhead = 4;                      // tiles from a dK/dV CTA's load to its prefetch

struct BwdParams {
  int L, L_kv;
  int batch, heads, kv_heads, heads_per_kv;
  int q_tiles, kv_tiles;
  unsigned dkdv_ctas;  // CTAs [0, dkdv_ctas) make dK and dV, the rest dQ
  int dkdv_splits, dq_splits;  // CTAs that share a tile's sum
  float *dkdv_parts, *dq_parts;  // fp32 [tile][split][dV, dK][128][128], [tile][split][128][128] (splits > 1)
  int causal_block;
  float scale, scale_log2;
  const int* q_lengths;
  const int* kv_lengths;
  const float* stats;  // [batch][heads][q_tiles][2][128]
  __nv_bfloat16 *dq, *dk, *dv;
  int64_t dq_stride_b, dq_stride_t, dk_stride_b, dk_stride_t, dv_stride_b, dv_stride_t;
};

// Which tile CTA `idx` of a role makes.  The tiles of a head follow one another, so that CTAs which run together share its
// operands in L2; causal sums differ in length, and there the longest of all heads come first.
struct TileOf {
  int at, head, batch;  // at: counted from the longest sum
  __device__ __forceinline__ TileOf(const BwdParams& p, unsigned idx, int tiles, int heads) {
    const unsigned sums = p.causal_block > 0 ? heads * p.batch : tiles;
    const int lo = static_cast<int>(idx % sums), hi = static_cast<int>(idx / sums);
    at = p.causal_block > 0 ? hi : lo;
    const int bh = p.causal_block > 0 ? lo : hi;
    head = bh % heads;
    batch = bh / heads;
  }
};

struct BwdShared {
  uint64_t fixed_full[2];                          // the operands a CTA keeps, for S and for dP: K and V, or Q and dO
  uint64_t a_full[DQ_K_STAGES], a_empty[DQ_K_STAGES];  // Q and statistics (dK/dV), K (dQ)
  uint64_t b_full[B_STAGES], b_empty[B_STAGES];        // dO (dK/dV), V (dQ)
  uint64_t zero_request, zeroed;  // the MMA issuer asks warp 2 to zero rows past the sequence's length; its answer
  uint64_t s_full[2], p_full[2], dp_full, dp_read, ds_full[2];  // p_full: dK/dV, by halves of the queries
  uint64_t dv_done, done;
  uint32_t tmem_base;
  int abort;
};

// D[128 x 128] (+)= A B^T, both tiles in shared memory with the 128 columns of d as the summed axis.
__device__ __forceinline__ void mma_tile_ss(uint32_t d, uint32_t a, uint32_t b) {
  constexpr uint32_t idesc = make_idesc(1, 1, 0, 0, BT, BT);
#pragma unroll
  for (int kk = 0; kk < HD / 16; ++kk) {
    const uint32_t off = (kk >> 2) * T_HALF_BYTES + (kk & 3) * 32;
    mma_f16_ss(d, make_sdesc_sw128(a + off, 16, 1024), make_sdesc_sw128(b + off, 16, 1024), idesc, kk > 0 ? 1u : 0u);
  }
}

// D[128 x 128] (+)= A B, steps [FIRST, LAST) of 16 of the summed axis: A (bf16, 128 x 128) in tensor memory, each
// run of RUN columns packed over the start of the RUN fp32 columns it came from; B's rows are the summed axis.
template <int RUN, int FIRST, int LAST>
__device__ __forceinline__ void mma_tile_ts(uint32_t d, uint32_t a, uint32_t b, bool accumulate) {
  constexpr uint32_t idesc = make_idesc(1, 1, 0, 1, BT, HD);
#pragma unroll
  for (int kk = FIRST; kk < LAST; ++kk)
    mma_f16_ts(d, a + kk * 16 / RUN * RUN + kk * 16 % RUN / 2, make_sdesc_sw128(b + kk * 2048, T_HALF_BYTES, 1024), idesc,
               (accumulate || kk > 0) ? 1u : 0u);
}

// `columns` fp32 columns of a warp's 32 rows to a CTA's part of a shared sum (rows of 128, a row per lane).
__device__ __forceinline__ void store_part(uint32_t taddr, int columns, float* dst, uint32_t lane) {
#pragma unroll 1
  for (int oc = 0; oc < columns / 32; ++oc) {
    uint32_t r[32];
    tmem_ld32(taddr + oc * 32, r);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 8; ++i)
      reinterpret_cast<uint4*>(dst + lane * HD + oc * 32)[i] =
          make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
  }
}

// A group's 64 columns of a gradient tile (a row per thread), by a TMA store from `half`, a half tile of shared memory
// that nothing else uses any more.  All 128 threads come here, those whose wait failed included.
__device__ __forceinline__ void store_half(uint32_t taddr, float scale, uint8_t* half, const CUtensorMap* map, int g,
                                           uint32_t row, int head, int row0, int batch, bool ok) {
  if (ok) stage_row64(taddr, scale, false, half, row);
  fence_async_shared();
  named_bar_sync(1 + g, 128);
  if (row == 0 && ok) {
    tma_store_4d(map, half, g * 64, head, row0, batch);
    tma_store_commit();
    tma_store_wait_read();
  }
}

// One arrival for the warp's tensor-memory accesses so far (32 would queue at the barrier).
__device__ __forceinline__ void warp_arrive(uint64_t* bar, uint32_t lane) {
  tc_fence_before();
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
}

__device__ __forceinline__ void zero_row(__nv_bfloat16* dst, int columns) {
  for (int i = 0; i < columns / 8; ++i) reinterpret_cast<uint4*>(dst)[i] = make_uint4(0, 0, 0, 0);
}

// ex2_poly2 whose power of two is a factor: added to the bits of a NaN, as there, it would make a finite number of it.
__device__ __forceinline__ f2 ex2_poly2_nan(f2 x) {
  const f2 magic{12583039.0f, 12583039.0f};  // 1.5 * 2^23 and the exponent's bias
  x.x = max_nan(x.x, -126.0f);
  x.y = max_nan(x.y, -126.0f);
  const f2 t = add2(x, magic);
  const f2 f = sub2(x, sub2(t, magic));
  f2 p = fma2(f2{0.0551716648f, 0.0551716648f}, f, f2{0.2426111251f, 0.2426111251f});
  p = fma2(p, f, f2{0.6932609677f, 0.6932609677f});
  p = fma2(p, f, f2{0.9999280572f, 0.9999280572f});
  return mul2(p, f2{__int_as_float(__float_as_int(t.x) << 23), __int_as_float(__float_as_int(t.y) << 23)});
}

// 32 scores of a row to probabilities: exp2(score * c + offset), three quarters on the MUFU and one on the FMA pipe.
// offset(i): the offsets of columns i .. i + 3.
template <typename Offset>
__device__ __forceinline__ void probabilities(float* s, float c, Offset offset) {
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    const float4 o = offset(i);
    const bool poly = i >= 24;
    const f2 a = fma2(f2{s[i], s[i + 1]}, f2{c, c}, f2{o.x, o.y});
    const f2 b = fma2(f2{s[i + 2], s[i + 3]}, f2{c, c}, f2{o.z, o.w});
    const f2 pa = poly ? ex2_poly2_nan(a) : f2{ex2(a.x), ex2(a.y)};
    const f2 pb = poly ? ex2_poly2_nan(b) : f2{ex2(b.x), ex2(b.y)};
    s[i] = pa.x;
    s[i + 1] = pa.y;
    s[i + 2] = pb.x;
    s[i + 3] = pb.y;
  }
}

// 32 values as bf16 over the start of the tensor-memory columns at taddr.
__device__ __forceinline__ void store_packed(uint32_t taddr, const float* v) {
  uint32_t pk[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) pk[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
  tmem_st16(taddr, pk);
}

// ------------------------------------------------------------------------------------------- row statistics
// 16 lanes per (token, head) row; a team of such groups takes the heads of 8 tokens, so that a group's statistics of a
// head leave as two whole 32-byte sectors (4-byte pieces of 16 sectors took 40 us at 9216 x 32 rows, this 27).
// Rows past the sequence's length, rows that saw no key and the tiles' padding rows get -lse = -inf, so their
// probabilities are 0.
struct StatsParams {
  const __nv_bfloat16 *dout, *out;
  int64_t dout_stride_b, dout_stride_t, out_stride_b, out_stride_t;
  const float* lse;
  const int* q_lengths;
  float* stats;
  int L, heads, q_tiles;
  int team;  // groups per 8 tokens, a power of two
};
constexpr int kStatsTokens = 8;

__global__ void __launch_bounds__(256, 4) attn_bwd_stats_kernel(StatsParams p) {
  pdl_trigger();
  pdl_wait();
  const int sub = threadIdx.x & 15;
  const int group = threadIdx.x >> 4;
  const int member = group & (p.team - 1);
  const int batch = blockIdx.y;
  const int token0 = (static_cast<int>(blockIdx.x) * (16 / p.team) + group / p.team) * kStatsTokens;
  if (token0 - group / p.team * kStatsTokens >= p.q_tiles * BT) return;  // the whole CTA lies past the last tile
  const int live = clamp_length(p.q_lengths, batch, p.L);
  const int mine = token0 + (sub & 7);  // the token whose statistics this lane writes: -lse (lanes 0-7), -delta (8-15)
  const __nv_bfloat16* dout = p.dout + batch * p.dout_stride_b + sub * 8;
  const __nv_bfloat16* out = p.out + batch * p.out_stride_b + sub * 8;
  // whole warps run every iteration: the reduction names all lanes
  for (int h0 = 0; h0 < p.heads; h0 += p.team) {
    const int head = h0 + member;
    const bool ok = head < p.heads;
    const float lse = ok && mine < live ? p.lse[(static_cast<int64_t>(batch) * p.heads + head) * p.L + mine] : -INFINITY;
    float delta = 0.f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint4 a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int token = token0 + half * 4 + i;
        a[i] = b[i] = make_uint4(0, 0, 0, 0);
        if (ok && token < live) {
          a[i] = __ldcs(reinterpret_cast<const uint4*>(dout + token * p.dout_stride_t + head * HD));
          b[i] = __ldcs(reinterpret_cast<const uint4*>(out + token * p.out_stride_t + head * HD));
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x[8], y[8], d = 0.f;
        unpack8(a[i], x);
        unpack8(b[i], y);
#pragma unroll
        for (int e = 0; e < 8; ++e) d = fmaf(x[e], y[e], d);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        if ((sub & 7) == half * 4 + i) delta = d;
      }
    }
    if (ok && mine < p.q_tiles * BT) {
      const bool empty = lse == -INFINITY;
      float* dst = p.stats + ((static_cast<int64_t>(batch) * p.heads + head) * p.q_tiles + mine / BT) * STAT_FLOATS + mine % BT;
      if (sub < 8)
        dst[0] = empty ? -INFINITY : -lse * 1.4426950408889634f;
      else
        dst[BT] = empty ? 0.f : -delta;
    }
  }
}

// ------------------------------------------------------------------------------------------- dK and dV
// One tile of 128 keys; keys are the rows (TMEM lanes) of every product, so P^T and dS^T feed the dV and dK
// products from tensor memory and a softmax thread owns one key.
//   TMEM: S^T [0,128), dP^T [128,256), dV [256,384), dK [384,512); bf16 P^T over S^T, dS^T over dP^T.
// Per query tile the MMA issuer runs dV += P dO, S(next), dK += dS Q, dP(next): while the softmax groups turn S
// into P the tensor pipe does the previous tile's dK and this tile's dP, and while they turn dP into dS it does
// dV and the next S.  A group of four warps takes 32 query columns of the first half and 32 of the second, and P goes
// to the MMA issuer half by half: the first half's dV runs while the second half is still exponentials.
__device__ __forceinline__ void bwd_dkdv(const CUtensorMap* tq, const CUtensorMap* tk, const CUtensorMap* tv,
                                         const CUtensorMap* tdo, const CUtensorMap* tdk, const CUtensorMap* tdv,
                                         const BwdParams& p, BwdShared& st, uint8_t* smem, uint32_t tmem) {
  uint8_t* k_tile = smem;
  uint8_t* v_tile = smem + T_BYTES;
  uint8_t* q_tiles = smem + 2 * T_BYTES;
  uint8_t* do_tiles = q_tiles + B_STAGES * T_BYTES;
  uint8_t* stat_tiles = do_tiles + B_STAGES * T_BYTES;
  const uint32_t warp = warp_idx();
  const uint32_t lane = threadIdx.x & 31;
  volatile int* abort = &st.abort;

  const int split = static_cast<int>(blockIdx.x % p.dkdv_splits);
  const unsigned idx = blockIdx.x / p.dkdv_splits;
  const TileOf own(p, idx, p.kv_tiles, p.kv_heads);
  const int kv_head = own.head;
  const int batch = own.batch;
  const int k0 = own.at * BT;  // the first keys are seen by the most queries
  const Visibility vis{clamp_length(p.q_lengths, batch, p.L), clamp_length(p.kv_lengths, batch, p.L_kv),
                       p.causal_block, p.L_kv - p.L};
  const int first_tile = max(vis.first(k0), 0) / BT;
  const int end_tile = (vis.q_len + BT - 1) / BT;
  const int per_head = (k0 >= vis.kv_len || end_tile <= first_tile) ? 0 : end_tile - first_tile;
  // this CTA's tiles of all those of the group's heads: [begin, begin + n)
  const int all = per_head * p.heads_per_kv;
  const int share = (all + p.dkdv_splits - 1) / p.dkdv_splits;
  const int begin = min(split * share, all);
  const int n = min(share, all - begin);
  const int head0 = kv_head * p.heads_per_kv + (per_head > 0 ? begin / per_head : 0);
  const int tile0 = first_tile + (per_head > 0 ? begin % per_head : 0);
  float* part = p.dkdv_parts + (static_cast<int64_t>(idx) * p.dkdv_splits + split) * (2 * BT * HD);
  // Rows that hold the caller's memory, whatever that is: those past the sequence's length in each head's last query
  // tile, and in its first one those that causality leaves without keys (more queries than keys).  0 * NaN in the dV and
  // dK products, which sum over these rows, would reach every key, so warp 2 zeroes them.
  const int tail = vis.q_len < p.L ? vis.q_len % BT : 0;  // the first row past the length, 0: none in the tile
  const int blind = p.causal_block > 0 ? max(-vis.shift - first_tile * BT, 0) : 0;  // rows [0, blind) see no key
  const auto zeroes = [&](int j) {  // whether this CTA's tile j has such rows
    if (tail == 0 && blind == 0) return false;
    const int at = (begin + j) % per_head;
    return (blind > 0 && at == 0) || (tail > 0 && at == per_head - 1);
  };

  if (n == 0) {
    if (warp >= 4 && p.dkdv_splits > 1) {
      for (int i = threadIdx.x - 128; i < 2 * BT * HD / 4; i += 256)
        reinterpret_cast<uint4*>(part)[i] = make_uint4(0, 0, 0, 0);
    } else if (warp >= 4) {
      const int key = k0 + static_cast<int>((warp & 3) * 32 + lane);
      const int64_t column = static_cast<int64_t>(kv_head) * HD;
      if (key < p.L_kv)
        zero_row(warp < 8 ? p.dv + batch * p.dv_stride_b + key * p.dv_stride_t + column
                          : p.dk + batch * p.dk_stride_b + key * p.dk_stride_t + column,
                 HD);
    }
    return;
  }

  if (warp == 0) {
    if (elect_one()) {
      // ---------------------------------------------------------- TMA producer
      mbar_arrive_expect_tx(&st.fixed_full[0], T_BYTES);
      load_rows(k_tile, tk, &st.fixed_full[0], T_HALF_BYTES, kv_head, k0, batch);
      int a_issued = 0, b_issued = 0;
      int head = head0, tile = tile0;
      // The ring holds two tiles, too few where they come from HBM.  So they are brought to L2 four tiles ahead, each by
      // one of the CTAs that share them (9216 x 1000, 32 heads: 468 us without, 464 with; 2304 x 2304 246 and 240).
      const int sharers = min(p.kv_tiles, 8), turn = own.at % sharers;
      int ahead_head = head0, ahead = tile0;
      for (int j = 0; j < n; ++j) {
        const int s = j % B_STAGES;
        const uint32_t ph = (j / B_STAGES) & 1;
        if (!mbar_wait(&st.a_empty[s], ph ^ 1u, abort)) break;
        mbar_arrive_expect_tx(&st.a_full[s], T_BYTES + STAT_BYTES);
        load_rows(q_tiles + s * T_BYTES, tq, &st.a_full[s], T_HALF_BYTES, head, tile * BT, batch);
        rows::bulk_load(stat_tiles + s * STAT_BYTES,
                        p.stats + ((static_cast<int64_t>(batch) * p.heads + head) * p.q_tiles + tile) * STAT_FLOATS,
                        STAT_BYTES, &st.a_full[s]);
        ++a_issued;
        if (j == 0) {  // behind what the first scores need
          mbar_arrive_expect_tx(&st.fixed_full[1], T_BYTES);
          load_rows(v_tile, tv, &st.fixed_full[1], T_HALF_BYTES, kv_head, k0, batch);
        }
        if (!mbar_wait(&st.b_empty[s], ph ^ 1u, abort)) break;
        mbar_arrive_expect_tx(&st.b_full[s], T_BYTES);
        load_rows(do_tiles + s * T_BYTES, tdo, &st.b_full[s], T_HALF_BYTES, head, tile * BT, batch);
        ++b_issued;
        if (++tile == end_tile) {
          tile = first_tile;
          ++head;
        }
        for (int i = j == 0 ? 0 : j + kAhead; i <= j + kAhead && i < n; ++i) {
          if (i > 1 && ahead % sharers == turn) {
            for (int h = 0; h < 2; ++h) {
              tma_prefetch_4d(tq, h * 64, ahead_head, ahead * BT, batch);
              tma_prefetch_4d(tdo, h * 64, ahead_head, ahead * BT, batch);
            }
          }
          if (++ahead == end_tile) {
            ahead = first_tile;
            ++ahead_head;
          }
        }
      }
      if (*abort) {  // let the copies in flight land before the CTA exits
        mbar_wait(&st.fixed_full[0], 0, nullptr);
        if (a_issued > 0) mbar_wait(&st.fixed_full[1], 0, nullptr);
        for (int j = a_issued - 1; j >= 0 && j >= a_issued - B_STAGES; --j)
          mbar_wait(&st.a_full[j % B_STAGES], (j / B_STAGES) & 1, nullptr);
        for (int j = b_issued - 1; j >= 0 && j >= b_issued - B_STAGES; --j)
          mbar_wait(&st.b_full[j % B_STAGES], (j / B_STAGES) & 1, nullptr);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      // ---------------------------------------------------------- MMA issuer
      const uint32_t t_s = tmem, t_dp = tmem + 128, t_dv = tmem + 256, t_dk = tmem + 384;
      const uint32_t k_addr = smem_u32(k_tile), v_addr = smem_u32(v_tile);
      const uint32_t q_addr = smem_u32(q_tiles), do_addr = smem_u32(do_tiles);
      uint32_t requests = 0;
      // Q of tile j in shared memory, the rows of Q and dO that hold anything zeroed
      auto q_ready = [&](int j) {
        const int s = j % B_STAGES;
        if (!mbar_wait(&st.a_full[s], (j / B_STAGES) & 1, abort)) return false;
        if (zeroes(j)) {
          if (!mbar_wait(&st.b_full[s], (j / B_STAGES) & 1, abort)) return false;
          mbar_arrive(&st.zero_request);
          if (!mbar_wait(&st.zeroed, requests++ & 1, abort)) return false;
        }
        tc_fence_after();
        return true;
      };
      auto issue_s = [&](int j) {
        mma_tile_ss(t_s, k_addr, q_addr + (j % B_STAGES) * T_BYTES);
        mma_commit(&st.s_full[0]);
      };
      auto issue_dp = [&](int j) {
        mma_tile_ss(t_dp, v_addr, do_addr + (j % B_STAGES) * T_BYTES);
        mma_commit(&st.dp_full);
      };
      bool ok = mbar_wait(&st.fixed_full[0], 0, abort) && q_ready(0);
      if (ok) issue_s(0);
      ok = ok && mbar_wait(&st.fixed_full[1], 0, abort) && mbar_wait(&st.b_full[0], 0, abort);
      if (ok) {
        tc_fence_after();
        issue_dp(0);
      }
      for (int j = 0; j < n && ok; ++j) {
        const int s = j % B_STAGES;
        if (!mbar_wait(&st.p_full[0], j & 1, abort)) break;
        tc_fence_after();
        mma_tile_ts<32, 0, 4>(t_dv, t_s, do_addr + s * T_BYTES, j > 0);
        if (!mbar_wait(&st.p_full[1], j & 1, abort)) break;
        tc_fence_after();
        mma_tile_ts<32, 4, 8>(t_dv, t_s, do_addr + s * T_BYTES, true);
        mma_commit(&st.b_empty[s]);
        if (j + 1 == n) mma_commit(&st.dv_done);
        if (j + 1 < n) {
          if (!q_ready(j + 1)) break;
          issue_s(j + 1);
        }
        if (!mbar_wait(&st.ds_full[0], j & 1, abort)) break;
        tc_fence_after();
        mma_tile_ts<32, 0, 8>(t_dk, t_dp, q_addr + s * T_BYTES, j > 0);
        mma_commit(&st.a_empty[s]);
        if (j + 1 < n) {
          const int s1 = (j + 1) % B_STAGES;
          if (!mbar_wait(&st.b_full[s1], ((j + 1) / B_STAGES) & 1, abort)) break;
          tc_fence_after();
          issue_dp(j + 1);
        }
      }
      mma_commit(&st.done);
      mbar_wait(&st.done, 0, nullptr);
    }
  } else if (warp == 2) {
    if (tail > 0 || blind > 0) {
      // ---------------------------------------------------------- zeroes the query rows that hold anything
      uint32_t request = 0;
      for (int j = 0; j < n; ++j) {
        if (!zeroes(j)) continue;
        const int s = j % B_STAGES;
        const uint32_t ph = (j / B_STAGES) & 1;
        if (!mbar_wait(&st.zero_request, request++ & 1, abort, kSumWaitLimitNs)) break;
        if (!mbar_wait(&st.a_full[s], ph, abort) || !mbar_wait(&st.b_full[s], ph, abort)) break;
        const int at = (begin + j) % per_head;
        for (uint8_t* tile : {q_tiles + s * T_BYTES, do_tiles + s * T_BYTES}) {
          if (at == 0) zero_rows(tile, T_HALF_BYTES, 0, blind, lane);
          if (tail > 0 && at == per_head - 1) zero_rows(tile, T_HALF_BYTES, tail, BT, lane);
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&st.zeroed);
      }
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax groups
    const int g = static_cast<int>(warp - 4) >> 2;  // query columns [32g, 32g + 32) and 64 on
    const uint32_t quarter = warp & 3;
    const int key = k0 + static_cast<int>(quarter * 32 + lane);
    const uint32_t lane_off = (quarter * 32u) << 16;
    const uint32_t s_tmem = tmem + lane_off + g * 32;
    const uint32_t dp_tmem = s_tmem + 128;
    const bool key_ok = key < vis.kv_len;
    const int first = vis.first(key);
    // every key row of the tile sees the queries from here on
    const int all_from = vis.first(min(k0 + BT, vis.kv_len) - 1);
    const bool ragged_keys = k0 + BT > vis.kv_len;
    bool ok = true;
    int tile = tile0;
    for (int j = 0; j < n; ++j) {
      const int s = j % B_STAGES;
      const int q0 = tile * BT;
      if (++tile == end_tile) tile = first_tile;
      const bool masked = ragged_keys || q0 < all_from || q0 + BT > vis.q_len;
      const int lo = key_ok ? first - q0 - g * 32 : BT;  // columns from this thread's first that its key is seen by
      const int hi = vis.q_len - q0 - g * 32;
      const float* stat = reinterpret_cast<const float*>(stat_tiles + s * STAT_BYTES) + g * 32;
      if (!mbar_wait(&st.a_full[s], (j / B_STAGES) & 1, abort) || !mbar_wait(&st.s_full[0], j & 1, abort)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float pr[64];
      tmem_ld32(s_tmem, *reinterpret_cast<uint32_t(*)[32]>(&pr[0]));
      tmem_ld32(s_tmem + 64, *reinterpret_cast<uint32_t(*)[32]>(&pr[32]));
      tmem_ld_wait();
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        probabilities(pr + half * 32, p.scale_log2,
                      [&](int i) { return *reinterpret_cast<const float4*>(stat + half * 64 + i); });
        if (masked) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (half * 64 + i < lo || half * 64 + i >= hi) pr[half * 32 + i] = 0.f;
        }
        store_packed(s_tmem + half * 64, pr + half * 32);
        tmem_st_wait();
        warp_arrive(&st.p_full[half], lane);
      }

      if (!mbar_wait(&st.dp_full, j & 1, abort)) {
        ok = false;
        break;
      }
      tc_fence_after();
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float dp[32];
        tmem_ld32(dp_tmem + half * 64, *reinterpret_cast<uint32_t(*)[32]>(&dp[0]));
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const int c = half * 32 + i;
          const float4 nd = *reinterpret_cast<const float4*>(stat + BT + half * 64 + i);
          const f2 x = mul2(f2{pr[c], pr[c + 1]}, add2(f2{dp[i], dp[i + 1]}, f2{nd.x, nd.y}));
          const f2 y = mul2(f2{pr[c + 2], pr[c + 3]}, add2(f2{dp[i + 2], dp[i + 3]}, f2{nd.z, nd.w}));
          dp[i] = x.x;
          dp[i + 1] = x.y;
          dp[i + 2] = y.x;
          dp[i + 3] = y.y;
        }
        if (masked) {  // dP of a masked pair may be anything
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (half * 64 + i < lo || half * 64 + i >= hi) dp[i] = 0.f;
        }
        store_packed(dp_tmem + half * 64, dp);
      }
      tmem_st_wait();
      warp_arrive(&st.ds_full[0], lane);
    }
    // each group stores half of the columns of both: dV while the last dK product runs, then dK
    const uint32_t row = quarter * 32 + lane;
    ok = ok && mbar_wait(&st.dv_done, 0, abort);
    tc_fence_after();
    if (p.dkdv_splits == 1)
      store_half(tmem + lane_off + 256 + g * 64, 1.f, do_tiles + g * T_HALF_BYTES, tdv, g, row, kv_head, k0, batch, ok);
    else if (ok)
      store_part(tmem + lane_off + 256 + g * 64, 64, part + quarter * 32 * HD + g * 64, lane);
    ok = ok && mbar_wait(&st.done, 0, abort);
    tc_fence_after();
    if (p.dkdv_splits == 1)
      store_half(tmem + lane_off + 384 + g * 64, p.scale, q_tiles + g * T_HALF_BYTES, tdk, g, row, kv_head, k0, batch, ok);
    else if (ok)
      store_part(tmem + lane_off + 384 + g * 64, 64, part + BT * HD + quarter * 32 * HD + g * 64, lane);
  }
}

// ------------------------------------------------------------------------------------------- dQ
// One tile of 128 queries; a softmax thread owns one query, so its statistics are two registers.
//   TMEM: S in two buffers [0,128) [128,256), dP [256,384), dQ [384,512); bf16 dS over its S buffer.
// P never leaves the registers here.  With two score buffers S(j+1) is ready before the softmax of tile j ends,
// and dP(j+1) runs as soon as dP(j) is in registers.
__device__ __forceinline__ void bwd_dq(const CUtensorMap* tq, const CUtensorMap* tk, const CUtensorMap* tv,
                                       const CUtensorMap* tdo, const CUtensorMap* tdq, const BwdParams& p,
                                       BwdShared& st, uint8_t* smem, uint32_t tmem) {
  uint8_t* q_tile = smem;
  uint8_t* do_tile = smem + T_BYTES;
  uint8_t* k_tiles = smem + 2 * T_BYTES;
  uint8_t* v_tiles = k_tiles + DQ_K_STAGES * T_BYTES;
  const uint32_t warp = warp_idx();
  const uint32_t lane = threadIdx.x & 31;
  volatile int* abort = &st.abort;

  const int split = static_cast<int>((blockIdx.x - p.dkdv_ctas) % p.dq_splits);
  const unsigned idx = (blockIdx.x - p.dkdv_ctas) / p.dq_splits;
  const TileOf own(p, idx, p.q_tiles, p.heads);
  const int head = own.head;
  const int batch = own.batch;
  const int kv_head = head / p.heads_per_kv;
  const int q0 = (p.q_tiles - 1 - own.at) * BT;  // causal rows get longer with their index
  const Visibility vis{clamp_length(p.q_lengths, batch, p.L), clamp_length(p.kv_lengths, batch, p.L_kv),
                       p.causal_block, p.L_kv - p.L};
  const int last = min(q0 + BT, vis.q_len) - 1;
  // this CTA's tiles of those its queries see: [tile0, tile0 + n)
  const int all = last < q0 ? 0 : (vis.limit(last) + BT - 1) / BT;
  const int share = (all + p.dq_splits - 1) / p.dq_splits;
  const int tile0 = min(split * share, all);
  const int n = min(share, all - tile0);
  const int border = vis.kv_len / BT - tile0;
  const int fix_tile = (vis.kv_len < p.L_kv && vis.kv_len % BT != 0 && border >= 0 && border < n) ? border : -1;
  float* part = p.dq_parts + (static_cast<int64_t>(idx) * p.dq_splits + split) * (BT * HD);

  if (n == 0) {
    if (warp >= 4 && p.dq_splits > 1) {
      for (int i = threadIdx.x - 128; i < BT * HD / 4; i += 256) reinterpret_cast<uint4*>(part)[i] = make_uint4(0, 0, 0, 0);
    } else if (warp >= 4) {
      const int token = q0 + static_cast<int>((warp & 3) * 32 + lane);
      if (token < p.L)
        zero_row(p.dq + batch * p.dq_stride_b + token * p.dq_stride_t + static_cast<int64_t>(head) * HD +
                     (warp < 8 ? 0 : 64),
                 64);
    }
    return;
  }

  if (warp == 0) {
    if (elect_one()) {
      // ---------------------------------------------------------- TMA producer
      mbar_arrive_expect_tx(&st.fixed_full[0], T_BYTES);
      load_rows(q_tile, tq, &st.fixed_full[0], T_HALF_BYTES, head, q0, batch);
      int a_issued = 0, b_issued = 0;
      for (int j = 0; j < n; ++j) {
        const int sk = j % DQ_K_STAGES, sv = j % B_STAGES;
        if (!mbar_wait(&st.a_empty[sk], ((j / DQ_K_STAGES) & 1) ^ 1u, abort)) break;
        mbar_arrive_expect_tx(&st.a_full[sk], T_BYTES);
        load_rows(k_tiles + sk * T_BYTES, tk, &st.a_full[sk], T_HALF_BYTES, kv_head, (tile0 + j) * BT, batch);
        ++a_issued;
        if (j == 0) {  // behind what the first scores need
          mbar_arrive_expect_tx(&st.fixed_full[1], T_BYTES);
          load_rows(do_tile, tdo, &st.fixed_full[1], T_HALF_BYTES, head, q0, batch);
        }
        if (!mbar_wait(&st.b_empty[sv], ((j / B_STAGES) & 1) ^ 1u, abort)) break;
        mbar_arrive_expect_tx(&st.b_full[sv], T_BYTES);
        load_rows(v_tiles + sv * T_BYTES, tv, &st.b_full[sv], T_HALF_BYTES, kv_head, (tile0 + j) * BT, batch);
        ++b_issued;
      }
      if (*abort) {  // let the copies in flight land before the CTA exits
        mbar_wait(&st.fixed_full[0], 0, nullptr);
        if (a_issued > 0) mbar_wait(&st.fixed_full[1], 0, nullptr);
        for (int j = a_issued - 1; j >= 0 && j >= a_issued - DQ_K_STAGES; --j)
          mbar_wait(&st.a_full[j % DQ_K_STAGES], (j / DQ_K_STAGES) & 1, nullptr);
        for (int j = b_issued - 1; j >= 0 && j >= b_issued - B_STAGES; --j)
          mbar_wait(&st.b_full[j % B_STAGES], (j / B_STAGES) & 1, nullptr);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      // ---------------------------------------------------------- MMA issuer
      const uint32_t t_dp = tmem + 256, t_dq = tmem + 384;
      const uint32_t q_addr = smem_u32(q_tile), do_addr = smem_u32(do_tile);
      const uint32_t k_addr = smem_u32(k_tiles), v_addr = smem_u32(v_tiles);
      auto issue_s = [&](int j) {
        if (!mbar_wait(&st.a_full[j % DQ_K_STAGES], (j / DQ_K_STAGES) & 1, abort)) return false;
        if (j == fix_tile) {
          mbar_arrive(&st.zero_request);
          if (!mbar_wait(&st.zeroed, 0, abort)) return false;
        }
        tc_fence_after();
        mma_tile_ss(tmem + (j & 1) * 128, q_addr, k_addr + (j % DQ_K_STAGES) * T_BYTES);
        mma_commit(&st.s_full[j & 1]);
        return true;
      };
      auto issue_dp = [&](int j) {
        if (!mbar_wait(&st.b_full[j % B_STAGES], (j / B_STAGES) & 1, abort)) return false;
        tc_fence_after();
        mma_tile_ss(t_dp, do_addr, v_addr + (j % B_STAGES) * T_BYTES);
        mma_commit(&st.dp_full);
        mma_commit(&st.b_empty[j % B_STAGES]);
        return true;
      };
      bool ok = mbar_wait(&st.fixed_full[0], 0, abort) && issue_s(0) && mbar_wait(&st.fixed_full[1], 0, abort) &&
                issue_dp(0) && (n < 2 || issue_s(1));
      for (int j = 0; j < n && ok; ++j) {
        if (j + 1 < n) {
          if (!mbar_wait(&st.dp_read, j & 1, abort)) break;
          if (!issue_dp(j + 1)) break;
        }
        if (!mbar_wait(&st.ds_full[j & 1], (j >> 1) & 1, abort)) break;
        tc_fence_after();
        mma_tile_ts<64, 0, 8>(t_dq, tmem + (j & 1) * 128, k_addr + (j % DQ_K_STAGES) * T_BYTES, j > 0);
        mma_commit(&st.a_empty[j % DQ_K_STAGES]);
        if (j + 2 < n && !issue_s(j + 2)) break;
      }
      mma_commit(&st.done);
      mbar_wait(&st.done, 0, nullptr);
    }
  } else if (warp == 2) {
    if (fix_tile >= 0) {
      // ---------------------------------------------------------- zeroes the K rows past the keys' length
      const int s = fix_tile % DQ_K_STAGES;
      if (mbar_wait(&st.zero_request, 0, abort, kSumWaitLimitNs) && mbar_wait(&st.a_full[s], (fix_tile / DQ_K_STAGES) & 1, abort)) {
        zero_rows(k_tiles + s * T_BYTES, T_HALF_BYTES, vis.kv_len % BT, BT, lane);
        fence_async_shared();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&st.zeroed);
    }
  } else if (warp >= 4) {
    // ------------------------------------------------------------ softmax groups
    const int g = static_cast<int>(warp - 4) >> 2;  // key columns [64g, 64g + 64)
    const uint32_t quarter = warp & 3;
    const int row = static_cast<int>(quarter * 32 + lane);
    const int token = q0 + row;
    const uint32_t lane_off = (quarter * 32u) << 16;
    const uint32_t dp_tmem = tmem + lane_off + 256 + g * 64;
    const float* stat =
        p.stats + ((static_cast<int64_t>(batch) * p.heads + head) * p.q_tiles + q0 / BT) * STAT_FLOATS + row;
    const float nl = stat[0], nd = stat[BT];
    const int limit = vis.limit(token);
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int b = j & 1;
      const uint32_t s_tmem = tmem + lane_off + b * 128 + g * 64;
      const int valid = limit - (tile0 + j) * BT - g * 64;  // columns of this thread's 64 that its query sees
      const bool masked = __any_sync(0xffffffffu, valid < 64);
      if (!mbar_wait(&st.s_full[b], (j >> 1) & 1, abort)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float pr[64];
      tmem_ld32(s_tmem, *reinterpret_cast<uint32_t(*)[32]>(&pr[0]));
      tmem_ld32(s_tmem + 32, *reinterpret_cast<uint32_t(*)[32]>(&pr[32]));
      tmem_ld_wait();
      probabilities(pr, p.scale_log2, [&](int) { return make_float4(nl, nl, nl, nl); });
      probabilities(pr + 32, p.scale_log2, [&](int) { return make_float4(nl, nl, nl, nl); });
      if (!mbar_wait(&st.dp_full, j & 1, abort)) {
        ok = false;
        break;
      }
      tc_fence_after();
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float dp[32];
        tmem_ld32(dp_tmem + half * 32, *reinterpret_cast<uint32_t(*)[32]>(&dp[0]));
        tmem_ld_wait();
        if (half == 1) {
          warp_arrive(&st.dp_read, lane);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int col = half * 32 + 2 * i;
          const f2 ds = mul2(f2{pr[col], pr[col + 1]}, add2(f2{dp[2 * i], dp[2 * i + 1]}, f2{nd, nd}));
          dp[2 * i] = ds.x;
          dp[2 * i + 1] = ds.y;
        }
        if (masked) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (half * 32 + i >= valid) dp[i] = 0.f;
        }
        store_packed(s_tmem + half * 16, dp);
      }
      tmem_st_wait();
      warp_arrive(&st.ds_full[b], lane);
    }
    ok = ok && mbar_wait(&st.done, 0, abort);
    tc_fence_after();
    if (p.dq_splits == 1)
      store_half(tmem + lane_off + 384 + g * 64, p.scale, q_tile + g * T_HALF_BYTES, tdq, g, row, head, q0, batch, ok);
    else if (ok)
      store_part(tmem + lane_off + 384 + g * 64, 64, part + quarter * 32 * HD + g * 64, lane);
  }
}

// Adds the parts of shared sums: a CTA per 32 rows of a tile (dV and dK tiles, then dQ tiles).
__global__ void __launch_bounds__(256) attn_bwd_join_kernel(const __grid_constant__ BwdParams p) {
  pdl_trigger();
  pdl_wait();
  const int col = (threadIdx.x & 31) * 4;  // a thread takes 4 columns of every eighth row
  const int row0 = (blockIdx.x & 3) * 32 + (threadIdx.x >> 5);
  const unsigned tile = blockIdx.x >> 2;
  const unsigned dkdv_tiles = p.dkdv_splits > 1 ? 2 * (p.dkdv_ctas / p.dkdv_splits) : 0;
  const float* src;
  __nv_bfloat16* dst;
  int64_t part_stride, row_stride;
  int splits, valid;
  float scale = p.scale;
  if (tile < dkdv_tiles) {
    const unsigned idx = tile >> 1;
    const bool is_dk = tile & 1;
    const TileOf own(p, idx, p.kv_tiles, p.kv_heads);
    const int k0 = own.at * BT, kv_head = own.head, batch = own.batch;
    splits = p.dkdv_splits;
    part_stride = 2 * BT * HD;
    src = p.dkdv_parts + static_cast<int64_t>(idx) * splits * part_stride + (is_dk ? BT * HD : 0);
    row_stride = is_dk ? p.dk_stride_t : p.dv_stride_t;
    dst = (is_dk ? p.dk + batch * p.dk_stride_b : p.dv + batch * p.dv_stride_b) + k0 * row_stride +
          static_cast<int64_t>(kv_head) * HD;
    valid = p.L_kv - k0;
    if (!is_dk) scale = 1.f;
  } else {
    const unsigned idx = tile - dkdv_tiles;
    const TileOf own(p, idx, p.q_tiles, p.heads);
    const int q0 = (p.q_tiles - 1 - own.at) * BT, head = own.head, batch = own.batch;
    splits = p.dq_splits;
    part_stride = BT * HD;
    src = p.dq_parts + static_cast<int64_t>(idx) * splits * part_stride;
    row_stride = p.dq_stride_t;
    dst = p.dq + batch * p.dq_stride_b + q0 * row_stride + static_cast<int64_t>(head) * HD;
    valid = p.L - q0;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = row0 + i * 8;
    if (row >= valid) continue;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < splits; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(src + k * part_stride + row * HD + col);
      sum.x += v.x;
      sum.y += v.y;
      sum.z += v.z;
      sum.w += v.w;
    }
    *reinterpret_cast<uint2*>(dst + row * row_stride + col) =
        make_uint2(pack_bf16x2(sum.x * scale, sum.y * scale), pack_bf16x2(sum.z * scale, sum.w * scale));
  }
}

__global__ void __launch_bounds__(kBwdThreads, 1)
    attn_bwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                    const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tdo,
                    const __grid_constant__ CUtensorMap tdq, const __grid_constant__ CUtensorMap tdk,
                    const __grid_constant__ CUtensorMap tdv, BwdParams p) {
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  __shared__ BwdShared st;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  const uint32_t warp = warp_idx();
  if (threadIdx.x == 0) {
    for (int s = 0; s < DQ_K_STAGES; ++s) {
      mbar_init(&st.a_full[s], 1);
      mbar_init(&st.a_empty[s], 1);
    }
    for (int s = 0; s < B_STAGES; ++s) {
      mbar_init(&st.b_full[s], 1);
      mbar_init(&st.b_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&st.fixed_full[b], 1);
      mbar_init(&st.s_full[b], 1);
      mbar_init(&st.p_full[b], kSoftmaxWarps);
      mbar_init(&st.ds_full[b], kSoftmaxWarps);
    }
    mbar_init(&st.dp_full, 1);
    mbar_init(&st.dp_read, kSoftmaxWarps);
    mbar_init(&st.zero_request, 1);
    mbar_init(&st.zeroed, 1);
    mbar_init(&st.dv_done, 1);
    mbar_init(&st.done, 1);
    st.abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&st.tmem_base, TMEM_COLS);
    tmem_relinquish();
  }
  pdl_wait();  // everything above touches only this CTA's shared memory and TMEM
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = st.tmem_base;
  if (blockIdx.x < p.dkdv_ctas)
    bwd_dkdv(&tq, &tk, &tv, &tdo, &tdk, &tdv, p, st, smem, tmem);
  else
    bwd_dq(&tq, &tk, &tv, &tdo, &tdq, p, st, smem, tmem);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

}  // namespace attn
}  // namespace ogx
