// Attention with softmax statistics, for the training pass: the dense kernel's arithmetic (attention.cuh) with per-batch
// lengths, a block-causal mask and shared key/value heads, and per row the log of the sum of the exponentials:
//   O = softmax(mask(c Q K^T)) V,  lse = log(sum exp(mask(c Q K^T))),  a row without keys: O = 0, lse = -inf.
//
// The roles and the tile loop are the dense kernel's: per CTA N tiles of 128 query rows, keys in tiles of 64, two score
// buffers per Q tile in tensor memory, P over its scores, O in tensor memory.  What differs is what surrounds the loop.
// With few keys (a prompt of 256: 4 tiles) a CTA of its own for every query block spends 12,000 cycles on starting,
// loading Q, its first scores and storing, against 1500 a tile.  So the CTAs stay, and take over blocks whose CTA has
// not started yet (cluster launch control): the next block's Q and first keys are loaded and its first scores are
// computed behind the last tiles of the current one, and a TMA store sends the output, staged in the block's Q tile,
// while the next block runs.  9216 x 256, 32 heads: 83 us with a CTA per block, 55 so; 2 x 2304 x 1024 91 and 76.
//   warp 0: TMA loads, and the next block   warp 1: MMA   warp 2: zeroes V's rows past the keys' length
//   warp 3: TMA stores                      warps 4..7 (and 8..11): softmax, a query row per thread
// At long sums the softmax sets the pace, as in the dense kernel: 9216 x 9216, 32 heads 1.14 ms = 1220 TFLOP/s, the tensor
// pipe active for 62 % of the cycles; causal by tokens 0.62 ms; 28,800 tokens, 4 heads, causal by 1800 0.77 ms.  These are
// the kernel's time in a burst of a few ms; back to back, under the 1000 W cap, 1.28, 0.71 and 0.86 ms.
// P is rounded to bf16, the type that the instruction wants where V is bf16: each term of O by 2^-8 at most, which leaves
// O 0.0021 to 0.0024 of its norm from the exact one where the rounding of O alone leaves 0.0017.  A second product with
// what the rounding dropped would cost half of the tensor work again.  The sum of the exponentials takes P unrounded.
// With N = 2 (one CTA per SM) each key tile is read once for 256 rows; with N = 1 (two CTAs per SM) fewer rows are
// wasted on an odd or single tile.
#pragma once

#include "attention.cuh"

namespace ogx {
namespace attn {

template <int N>
struct MaskedShape;
template <>
struct MaskedShape<2> {
  static constexpr int Q_BUFFERS = 2;  // the next block's Q arrives while this block's output leaves
  static constexpr int STAGES = 3;
  static constexpr int THREADS = kThreads;
  static constexpr int LAUNCH_REGS = kLaunchRegs;
  static constexpr uint32_t REGS_PRODUCER = kRegsProducer;
};
template <>
struct MaskedShape<1> {
  static constexpr int Q_BUFFERS = 1;
  static constexpr int STAGES = 2;
  static constexpr int THREADS = 256;
  static constexpr int LAUNCH_REGS = 128;
  static constexpr uint32_t REGS_PRODUCER = 56;
};
template <int N>
constexpr int kMaskedSmem =
    MaskedShape<N>::Q_BUFFERS * N * Q_TILE_BYTES + 2 * MaskedShape<N>::STAGES * KV_TILE_BYTES + 1024;
static_assert(128 * MaskedShape<1>::REGS_PRODUCER + 128 * kRegsSoftmax <=
                  MaskedShape<1>::THREADS * MaskedShape<1>::LAUNCH_REGS,
              "register split exceeds the launch");

struct MaskedParams {
  int L, L_kv;
  float scale_log2;  // softmax scale * log2(e)
  __nv_bfloat16* out;
  int64_t out_stride_b, out_stride_t;  // elements; the head stride is 128
  float* lse;                          // [batch, heads, L]: natural log of each row's sum of exponentials
  int heads;
  int heads_per_kv;       // query heads that share a key/value head
  int pack_shift;         // 2^pack_shift of these make a Q tile's rows together: row = token << pack_shift | head
  int causal_block;       // 0: every key is visible
  const int* q_lengths;   // [batch] or null
  const int* kv_lengths;  // [batch] or null
  // few query blocks over many keys: `splits` CTAs share a block's key tiles (split_tiles each) and leave their
  // unnormalised rows and row statistics, [batch][heads][splits][L] x (128 | max, sum), for attn_join_kernel
  unsigned splits;
  int split_tiles;
  float* part_o;
  float2* part_ml;
  unsigned blocks, head_groups;  // query blocks; heads >> pack_shift
  bool longest_first;  // the order of blocks
  bool one_wave;  // every block has a CTA that starts at once: there is none to take over
};

// Which keys a query sees.  Queries from q_len on see none; keys from kv_len on are seen by none.  With
// block > 0 the sequences end together: query i stands at position i + shift, shift = L_kv - L, and sees the
// keys of its own block of `block` positions and of all earlier blocks (block 1: the token-causal mask; the
// tokens of a latent frame: a frame-causal one).  Both forms below are prefixes, so a tile needs comparing
// only at its border.
struct Visibility {
  int q_len, kv_len, block, shift;
  // keys [0, limit) are visible to query i
  __device__ __forceinline__ int limit(int i) const {
    if (i >= q_len) return 0;
    if (block == 0) return kv_len;
    const int at = i + shift;
    if (at < 0) return 0;
    const int64_t end = static_cast<int64_t>(at) - at % block + block;
    return end < kv_len ? static_cast<int>(end) : kv_len;
  }
  // queries [first(j), q_len) see key j < kv_len
  __device__ __forceinline__ int first(int j) const { return block == 0 ? 0 : j - j % block - shift; }
};

__device__ __forceinline__ int clamp_length(const int* lengths, int batch, int full) {
  if (lengths == nullptr) return full;
  const int n = lengths[batch];
  return n < 0 ? 0 : (n > full ? full : n);
}

// Zeroes rows [row0, rows) of a tile of 128-byte rows (both 64-column halves) that a TMA load wrote, by one
// warp: rows past a sequence's length hold whatever the caller's memory holds there, and 0 * NaN in the
// product that sums over these rows would reach every output.  The caller has waited for the load and
// signals the MMA issuer afterwards.  (A 128-byte row stays its own 128 bytes under the swizzle.)
__device__ __forceinline__ void zero_rows(uint8_t* tile, int half_bytes, int row0, int rows, uint32_t lane) {
  for (int i = static_cast<int>(lane); i < (rows - row0) * 8; i += 32) {
    *reinterpret_cast<uint4*>(tile + row0 * 128 + i * 16) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(tile + half_bytes + row0 * 128 + i * 16) = make_uint4(0, 0, 0, 0);
  }
}

template <int N>
struct MaskedShared {
  static constexpr int STAGES = MaskedShape<N>::STAGES;
  uint4 next[2];  // launch control's answers
  uint64_t next_full[2], next_empty[2];
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[STAGES], k_empty[STAGES];
  uint64_t v_full[STAGES], v_empty[STAGES];
  uint64_t s_full[N][2];  // scores of tile q in buffer b are in TMEM
  uint64_t p_full[N][2];  // P of tile q in buffer b is in TMEM
  uint64_t o_ready[N];    // completes once per PV_q
  uint64_t o_done[N];     // a block's last PV_q completed
  uint64_t o_read[N];     // a block's O_q left tensor memory: staged in shared memory, or stored
  uint64_t drained;
  // The MMA issuer asks warp 2 to zero the rows past the keys in a block's last V tile, and its answer.  (A warp that
  // waited for that tile's load by parity alone could take an earlier load of the stage for it.)
  uint64_t v_fix_request, v_fixed;
  uint32_t tmem_base;
  int abort;
};

// Asks for the index of a CTA of this grid that has not started; it will not start then.  The 16-byte answer arrives at
// `bar`.  After an answer without an index there must be no further request.
__device__ __forceinline__ void request_next(uint4* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(answer)),
               "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ bool read_next(const uint4* answer, uint3* block) {
  uint32_t got;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
      "ld.shared.b128 r, [%4];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %3, 1, 0, p;\n\t"
      "mov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%0, %1, %2, _}, r;\n\t}\n"
      : "=r"(block->x), "=r"(block->y), "=r"(block->z), "=r"(got)
      : "r"(smem_u32(answer))
      : "memory");
  return got != 0;
}

// ex2_poly2 with a degree-4 polynomial (fitted in the same way, max relative error 2.7e-6) where the sum of the
// exponentials is itself a result: with the degree-3 one the statistics of short rows are 100 times further from
// exact than 32-bit arithmetic is.
__device__ __forceinline__ f2 ex2_poly2_sum(f2 x) {
  const f2 magic{12582912.0f, 12582912.0f};
  x.x = fmaxf(x.x, -126.0f);
  x.y = fmaxf(x.y, -126.0f);
  const f2 t = add2(x, magic);
  const f2 f = sub2(x, sub2(t, magic));
  f2 p = fma2(f2{0.0095701022f, 0.0095701022f}, f, f2{0.0559178591f, 0.0559178591f});
  p = fma2(p, f, f2{0.2402474433f, 0.2402474433f});
  p = fma2(p, f, f2{0.6931217909f, 0.6931217909f});
  p = fma2(p, f, f2{0.9999992847f, 0.9999992847f});
  return f2{__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)),
            __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23))};
}

// The running maximum of a row before its first score: the lowest finite one, so that scores of -inf add nothing.
constexpr float kNoScore = -3.40282347e38f;

// A thread's row of 64 fp32 columns in tensor memory, times `scale`, as bf16 into its place of a 64-column half tile
// that a TMA store takes (128-byte rows, 128-byte swizzle).  Stored straight from registers, every instruction would
// touch 32 rows: 4800 cycles for a 256-row block at 8 KB between rows; the staging takes 1700, and the store (2100, 30
// bytes per cycle and SM) needs no thread.
__device__ __forceinline__ void stage_row64(uint32_t taddr, float scale, bool zero, uint8_t* half, uint32_t row) {
#pragma unroll
  for (int oc = 0; oc < 2; ++oc) {
    uint32_t r[32];
    tmem_ld32(taddr + oc * 32, r);
    tmem_ld_wait();
#pragma unroll
    for (int v8 = 0; v8 < 4; ++v8) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = zero ? 0.f : __uint_as_float(r[v8 * 8 + i]) * scale;
      *reinterpret_cast<uint4*>(half + row * 128 + (((oc * 4 + v8) ^ (row & 7u)) << 4)) = pack8(f);
    }
  }
}

// A query block: where it lies and which key tiles this CTA multiplies with it.
template <int N>
struct Block {
  int head, batch, split, token0, tile0, nkv, fix_tile;
  Visibility vis;
  __device__ __forceinline__ Block(const MaskedParams& p, uint3 at) {
    const int tokens = (N * BQ) >> p.pack_shift;
    if (p.longest_first) {  // grid {split, head, batch | block}: longest rows, the last ones, first
      split = static_cast<int>(at.x % p.splits);
      const unsigned group = at.x / p.splits;
      head = static_cast<int>(group % p.head_groups);
      batch = static_cast<int>(group / p.head_groups);
      token0 = static_cast<int>(p.blocks - 1 - at.y) * tokens;
    } else {  // grid {block | head | split, batch}: the blocks of a head run together and share its keys in L2
      token0 = static_cast<int>(at.x) * tokens;
      head = static_cast<int>(at.y);
      split = static_cast<int>(at.z % p.splits);
      batch = static_cast<int>(at.z / p.splits);
    }
    head <<= p.pack_shift;  // the first of the group
    tile0 = split * p.split_tiles;
    vis = Visibility{clamp_length(p.q_lengths, batch, p.L), clamp_length(p.kv_lengths, batch, p.L_kv), p.causal_block,
                     p.L_kv - p.L};
    const int last = min(token0 + tokens, vis.q_len) - 1;  // limit() grows with the row
    nkv = last < token0 ? 0 : (vis.limit(last) + BKV - 1) / BKV;
    nkv = min(max(nkv - tile0, 0), p.split_tiles);
    const int border = vis.kv_len / BKV - tile0;
    // the V tile whose last rows lie past the keys' length
    fix_tile = vis.kv_len < p.L_kv && vis.kv_len % BKV != 0 && border >= 0 && border < nkv ? border : -1;
  }
};

template <int N>
__global__ void __launch_bounds__(MaskedShape<N>::THREADS, N == 2 ? 1 : 2)
    attn_masked_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                       const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tout,
                       const MaskedParams p) {
  constexpr int STAGES = MaskedShape<N>::STAGES;
  constexpr int QB = MaskedShape<N>::Q_BUFFERS;
  constexpr uint32_t T_S = 128 * N;  // TMEM: O tiles first, then two score buffers for each
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  __shared__ MaskedShared<N> st;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  // [Q buffers][K stages][V stages]
  uint8_t* q_tiles = smem;
  uint8_t* k_tiles = smem + QB * N * Q_TILE_BYTES;
  uint8_t* v_tiles = k_tiles + STAGES * KV_TILE_BYTES;
  const uint32_t warp = warp_idx();
  const uint32_t lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int b = 0; b < 2; ++b) {
      mbar_init(&st.next_full[b], 1);
      mbar_init(&st.next_empty[b], 3 + 4 * N);  // warps 1 to 3 and the softmax warps
      mbar_init(&st.q_full[b], 1);
      mbar_init(&st.q_empty[b], 1);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&st.k_full[s], 1);
      mbar_init(&st.k_empty[s], 1);
      mbar_init(&st.v_full[s], 1);
      mbar_init(&st.v_empty[s], 1);
    }
    for (int q = 0; q < N; ++q) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&st.s_full[q][b], 1);
        mbar_init(&st.p_full[q][b], 128);
      }
      mbar_init(&st.o_ready[q], 1);
      mbar_init(&st.o_done[q], 1);
      mbar_init(&st.o_read[q], 128);
    }
    mbar_init(&st.drained, 1);
    mbar_init(&st.v_fix_request, 1);
    mbar_init(&st.v_fixed, 1);
    st.abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&st.tmem_base, 256 * N);
    tmem_relinquish();
  }
  pdl_wait();  // everything above touches only this CTA's shared memory and TMEM
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = st.tmem_base;
  volatile int* abort = &st.abort;
  uint3 at = blockIdx;

  // The block after item `i`, for every warp but the producer's.
  auto advance = [&](int i) {
    if (p.one_wave) return false;
    if (!mbar_wait(&st.next_full[i & 1], (i >> 1) & 1, abort, kSumWaitLimitNs)) return false;
    const bool more = read_next(&st.next[i & 1], &at);
    __syncwarp();
    if (lane == 0) mbar_arrive(&st.next_empty[i & 1]);
    return more;
  };

  if (warp < 4) {
    reg_dealloc<MaskedShape<N>::REGS_PRODUCER>();
    if (warp == 0) {
      if (elect_one()) {
        // ---------------------------------------------------------- TMA producer
        int kn = 0, vn = 0, live = 0;  // loads of K and V tiles, blocks with any
        bool more = true;
        int item = 0;
        for (; more; ++item) {
          // The next block is asked for shortly before this one's last load and read behind it: early enough to hide
          // the answer, late enough to leave the last blocks to CTAs that end sooner.
          const int slot = item & 1;
          bool asked = false;
          auto ask = [&] {
            if (item >= 2 && !mbar_wait(&st.next_empty[slot], ((item >> 1) - 1) & 1, abort)) return false;
            fence_async_shared();
            mbar_arrive_expect_tx(&st.next_full[slot], 16);
            request_next(&st.next[slot], &st.next_full[slot]);
            return asked = true;
          };
          const Block<N> b(p, at);
          const int ask_at = p.one_wave ? -1 : max(b.nkv - 2, 0);
          bool ok = true;
          if (b.nkv > 0) {
            const int qb = live % QB;
            if (live >= QB) ok = mbar_wait(&st.q_empty[qb], (live / QB - 1) & 1, abort);
            if (ok) {
              mbar_arrive_expect_tx(&st.q_full[qb], N * Q_TILE_BYTES);
              for (int q = 0; q < N; ++q)
                load_rows(q_tiles + (qb * N + q) * Q_TILE_BYTES, &tq, &st.q_full[qb], Q_HALF_BYTES, b.head,
                          b.token0 + (q * BQ >> p.pack_shift), b.batch);
              ++live;
            }
            const int kv_head = b.head / p.heads_per_kv;
            for (int j = 0; j < b.nkv && ok; ++j) {
              if (j == ask_at && !(ok = ask())) break;
              const int ks = kn % STAGES;
              if (!(ok = mbar_wait(&st.k_empty[ks], ((kn / STAGES) & 1) ^ 1u, abort))) break;
              mbar_arrive_expect_tx(&st.k_full[ks], KV_TILE_BYTES);
              load_rows(k_tiles + ks * KV_TILE_BYTES, &tk, &st.k_full[ks], KV_HALF_BYTES, kv_head,
                        (b.tile0 + j) * BKV, b.batch);
              ++kn;
              if (!(ok = mbar_wait(&st.v_empty[ks], ((vn / STAGES) & 1) ^ 1u, abort))) break;
              mbar_arrive_expect_tx(&st.v_full[ks], KV_TILE_BYTES);
              load_rows(v_tiles + ks * KV_TILE_BYTES, &tv, &st.v_full[ks], KV_HALF_BYTES, kv_head,
                        (b.tile0 + j) * BKV, b.batch);
              ++vn;
            }
          }
          if (b.nkv == 0 && ask_at == 0) ok = ask();
          // after a failure, too: the answer must have landed before the CTA ends
          if (asked && !mbar_wait(&st.next_full[slot], (item >> 1) & 1, nullptr)) break;
          more = asked && ok && read_next(&st.next[slot], &at);
        }
        if (*abort) {
          // let the copies already in flight land before the CTA exits
          for (int i = live - 1; i >= 0 && i >= live - QB; --i) mbar_wait(&st.q_full[i % QB], (i / QB) & 1, nullptr);
          for (int i = kn - 1; i >= 0 && i >= kn - STAGES; --i)
            mbar_wait(&st.k_full[i % STAGES], (i / STAGES) & 1, nullptr);
          for (int i = vn - 1; i >= 0 && i >= vn - STAGES; --i)
            mbar_wait(&st.v_full[i % STAGES], (i / STAGES) & 1, nullptr);
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- MMA issuer
      constexpr uint32_t idesc_qk = make_idesc(1, 1, 0, 0, BQ, BKV);  // bf16, K-major A and B
      constexpr uint32_t idesc_pv = make_idesc(1, 1, 0, 1, BQ, HD);   // bf16, V is MN-major
      const uint32_t k_addr = smem_u32(k_tiles);
      const uint32_t v_addr = smem_u32(v_tiles);
      const bool leader = elect_one();
      int base = 0, live = 0, fixes = 0;  // tiles and live blocks so far
      int ks = 0, vs = 0;                 // stages of the next K and V tile
      uint32_t kph = 0, vph = 0;
      bool ok = true;
      for (int item = 0;; ++item) {
        const Block<N> b(p, at);
        if (leader && b.nkv > 0) {
          const uint32_t q_addr = smem_u32(q_tiles) + (live % QB) * (N * Q_TILE_BYTES);
          auto issue_s = [&](int q, int t) {  // S_q of tile t into score buffer t % 2
            const uint32_t qa = q_addr + q * Q_TILE_BYTES;
            const uint32_t ka = k_addr + ks * KV_TILE_BYTES;
            const uint32_t d = tmem + T_S + q * 128 + (t & 1) * 64;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk) {
              const uint32_t qoff = (kk >> 2) * Q_HALF_BYTES + (kk & 3) * 32;
              const uint32_t koff = (kk >> 2) * KV_HALF_BYTES + (kk & 3) * 32;
              mma_f16_ss(d, make_sdesc_sw128(qa + qoff, 16, 1024), make_sdesc_sw128(ka + koff, 16, 1024), idesc_qk,
                         kk > 0 ? 1u : 0u);
            }
            mma_commit(&st.s_full[q][t & 1]);
          };
          auto next_k = [&] {  // behind the last product with this K tile
            mma_commit(&st.k_empty[ks]);
            if (++ks == STAGES) {
              ks = 0;
              kph ^= 1;
            }
          };
          auto issue_pv = [&](int q, int t, bool first, bool last) {  // O_q += P_q V
            const uint32_t va = v_addr + vs * KV_TILE_BYTES;
            const uint32_t pa = tmem + T_S + q * 128 + (t & 1) * 64;
#pragma unroll
            for (int kk = 0; kk < BKV / 16; ++kk) {
              mma_f16_ts(tmem + q * 128, pa + kk * 8, make_sdesc_sw128(va + kk * 2048, KV_HALF_BYTES, 1024), idesc_pv,
                         (!first || kk > 0) ? 1u : 0u);
            }
            mma_commit(&st.o_ready[q]);
            if (last) mma_commit(&st.o_done[q]);
          };
          ok = mbar_wait(&st.q_full[live % QB], (live / QB) & 1, abort);
          // the scores of the first two key tiles
          for (int j = 0; j < 2 && j < b.nkv && ok; ++j) {
            if (!(ok = mbar_wait(&st.k_full[ks], kph, abort))) break;
            tc_fence_after();
            for (int q = 0; q < N; ++q) issue_s(q, base + j);
            next_k();
          }
          for (int j = 0; j < b.nkv && ok; ++j) {
            const int t = base + j;
            const uint32_t pph = (t >> 1) & 1;
            const bool more_s = j + 2 < b.nkv;
            if (!(ok = mbar_wait(&st.v_full[vs], vph, abort) && mbar_wait(&st.p_full[0][t & 1], pph, abort))) break;
            if (j == b.fix_tile) {
              mbar_arrive(&st.v_fix_request);
              if (!(ok = mbar_wait(&st.v_fixed, fixes++ & 1, abort))) break;
            }
            // the first product overwrites O, which the block before must have left
            if (j == 0 && live > 0 && !(ok = mbar_wait(&st.o_read[0], (live - 1) & 1, abort))) break;
            tc_fence_after();
            issue_pv(0, t, j == 0, j + 1 == b.nkv);
            if (more_s) {
              if (!(ok = mbar_wait(&st.k_full[ks], kph, abort))) break;
              tc_fence_after();
              issue_s(0, t + 2);
            }
            if constexpr (N > 1) {
              if (!(ok = mbar_wait(&st.p_full[N - 1][t & 1], pph, abort))) break;
              if (j == 0 && live > 0 && !(ok = mbar_wait(&st.o_read[N - 1], (live - 1) & 1, abort))) break;
              tc_fence_after();
              issue_pv(N - 1, t, j == 0, j + 1 == b.nkv);
            }
            mma_commit(&st.v_empty[vs]);
            if (++vs == STAGES) {
              vs = 0;
              vph ^= 1;
            }
            if (more_s) {
              if constexpr (N > 1) issue_s(N - 1, t + 2);
              next_k();
            }
          }
          base += b.nkv;
          ++live;
        }
        __syncwarp();
        if (!advance(item) || *abort) break;
      }
      if (leader) {
        mma_commit(&st.drained);
        mbar_wait(&st.drained, 0, nullptr);
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------- V's rows past the length
      int base = 0, fixes = 0;
      for (int item = 0;; ++item) {
        const Block<N> b(p, at);
        if (b.fix_tile >= 0) {
          const int t = base + b.fix_tile;
          if (mbar_wait(&st.v_fix_request, fixes & 1, abort, kSumWaitLimitNs) &&
              mbar_wait(&st.v_full[t % STAGES], (t / STAGES) & 1, abort)) {
            zero_rows(v_tiles + (t % STAGES) * KV_TILE_BYTES, KV_HALF_BYTES, b.vis.kv_len % BKV, BKV, lane);
            fence_async_shared();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&st.v_fixed);
          ++fixes;
        }
        base += b.nkv;
        if (!advance(item)) break;
      }
    } else {
      // ---------------------------------------------------------- TMA stores
      int live = 0;
      for (int item = 0;; ++item) {
        const Block<N> b(p, at);
        if (b.nkv > 0) {
          if (lane == 0) {
            const int qb = live % QB;
            bool ok = true;
            for (int q = 0; q < N; ++q) {
              ok = ok && mbar_wait(&st.o_read[q], live & 1, abort, kSumWaitLimitNs);
              const int token = b.token0 + (q * BQ >> p.pack_shift);
              if (!ok || p.splits > 1 || token >= p.L) continue;
              for (int h = 0; h < 2; ++h)
                tma_store_4d(&tout, q_tiles + (qb * N + q) * Q_TILE_BYTES + h * Q_HALF_BYTES, h * 64, b.head, token,
                             b.batch);
              tma_store_commit();
            }
            tma_store_wait_read();
            mbar_arrive(&st.q_empty[qb]);
          }
          __syncwarp();
          ++live;
        }
        if (!advance(item)) break;
      }
    }
  } else {
    reg_alloc<kRegsSoftmax>();
    // ------------------------------------------------------------ softmax + epilogue
    const int q = (warp - 4) >> 2;                // Q tile of this warpgroup
    const uint32_t quarter = warp & 3;            // TMEM lane quarter of this warp
    const uint32_t row = quarter * 32 + lane;     // row within the Q tile
    const uint32_t lane_off = (quarter * 32u) << 16;
    const uint32_t o_tmem = tmem + lane_off + q * 128;
    const float c = p.scale_log2;
    int base = 0, live = 0;
    bool ok = true;
    for (int item = 0;; ++item) {
      const Block<N> blk(p, at);
      const int nkv = blk.nkv;
      const int token = blk.token0 + static_cast<int>((q * BQ + row) >> p.pack_shift);
      const int row_head = blk.head + static_cast<int>(row & ((1u << p.pack_shift) - 1));
      const int64_t batch_head = static_cast<int64_t>(blk.batch) * p.heads + row_head;
      // visible keys from this CTA's first one on
      const int limit = blk.vis.limit(token) - blk.tile0 * BKV;
      float m_run = kNoScore;  // running max, already multiplied by c
      float l_run = 0.f;
      for (int j = 0; j < nkv; ++j) {
        const int t = base + j;
        const int b = t & 1;
        const uint32_t s_tmem = tmem + lane_off + T_S + q * 128 + b * 64;
        if (!mbar_wait(&st.s_full[q][b], (t >> 1) & 1, abort)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t sr[64];
        tmem_ld32(s_tmem, *reinterpret_cast<uint32_t(*)[32]>(&sr[0]));
        tmem_ld32(s_tmem + 32, *reinterpret_cast<uint32_t(*)[32]>(&sr[32]));
        tmem_ld_wait();
        float* sf = reinterpret_cast<float*>(sr);
        const int kv_valid = limit - j * BKV;
        if (__any_sync(0xffffffffu, kv_valid < BKV)) {
#pragma unroll
          for (int i = 0; i < BKV; ++i)
            if (i >= kv_valid) sf[i] = -INFINITY;
        }
        // row max: four independent chains of 3-input max
        float mq[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          float m = max_nan(sf[h * 16], sf[h * 16 + 15]);
#pragma unroll
          for (int i = 1; i < 15; i += 2) m = max3_nan(m, sf[h * 16 + i], sf[h * 16 + i + 1]);
          mq[h] = m;
        }
        const float m_tile = max3_nan(max_nan(mq[0], mq[1]), mq[2], mq[3]) * c;
        float alpha = 1.f;
        bool rescale = false;
        if (!(m_tile <= m_run + kRescaleThreshold)) {  // NaN, too, becomes the maximum, and stays it
          alpha = ex2(m_run - m_tile);  // 0 at a row's first score
          m_run = m_tile;
          rescale = j > 0;
        }
        f2 rowsum2{0.f, 0.f};
        const f2 c2{c, c};
        const f2 negm{-m_run, -m_run};
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          uint32_t pk[8];
          const bool poly = (kPolyChunkMask >> cc) & 1u;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const f2 a = fma2(f2{sf[cc * 16 + 2 * i], sf[cc * 16 + 2 * i + 1]}, c2, negm);
            const f2 pr = poly ? ex2_poly2_sum(a) : f2{ex2(a.x), ex2(a.y)};
            rowsum2 = add2(rowsum2, pr);
            pk[i] = pack_bf16x2(pr.x, pr.y);
          }
          // P chunk cc -> TMEM columns [8cc, 8cc+8) of this score buffer (all scores are in registers)
          asm volatile(
              "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(s_tmem + cc * 8),
              "r"(pk[0]), "r"(pk[1]), "r"(pk[2]), "r"(pk[3]), "r"(pk[4]), "r"(pk[5]), "r"(pk[6]), "r"(pk[7])
              : "memory");
        }
        l_run = l_run * alpha + (rowsum2.x + rowsum2.y);
        if (__any_sync(0xffffffffu, rescale)) {
          // O must hold PV_q(t-1) before it is rescaled.  o_ready completes once per PV_q; S_q(t) was issued after
          // PV_q(t-2), so it is at most one phase behind phase t-1 here.
          if (!mbar_wait(&st.o_ready[q], (t - 1) & 1, abort)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int oc = 0; oc < 4; ++oc) {
            uint32_t orr[32];
            tmem_ld32(o_tmem + oc * 32, orr);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) orr[i] = __float_as_uint(__uint_as_float(orr[i]) * alpha);
            tmem_st32(o_tmem + oc * 32, orr);
          }
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&st.p_full[q][b]);
      }
      if (nkv == 0) {
        if (token < p.L && p.splits > 1) {
          p.part_ml[(batch_head * p.splits + blk.split) * p.L + token] = make_float2(-INFINITY, 0.f);
        } else if (token < p.L) {
          uint4* dst = reinterpret_cast<uint4*>(p.out + static_cast<int64_t>(blk.batch) * p.out_stride_b +
                                                static_cast<int64_t>(token) * p.out_stride_t +
                                                static_cast<int64_t>(row_head) * HD);
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) dst[i] = make_uint4(0, 0, 0, 0);
          p.lse[batch_head * p.L + token] = -INFINITY;
        }
      } else if ((ok = ok && mbar_wait(&st.o_done[q], live & 1, abort))) {
        tc_fence_after();
        // A row without a key, or of scores of -inf alone (its sum is 0, and out 0 / 0); a row with a score of NaN or +inf
        // is NaN (inf - inf), the log of its sum NaN or +inf.
        if (limit <= 0 || m_run == kNoScore) m_run = -INFINITY;
        if (!(fabsf(m_run) < INFINITY)) l_run = NAN;
        if (p.splits > 1) {
          const int64_t at_row = (batch_head * p.splits + blk.split) * p.L + token;
          if (token < p.L) p.part_ml[at_row] = make_float2(m_run, limit <= 0 ? 0.f : l_run);
#pragma unroll 1
          for (int oc = 0; oc < 4; ++oc) {
            uint32_t orr[32];
            tmem_ld32(o_tmem + oc * 32, orr);
            tmem_ld_wait();
            if (token < p.L && limit > 0) {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                reinterpret_cast<uint4*>(p.part_o + at_row * HD + oc * 32)[i] =
                    make_uint4(orr[4 * i], orr[4 * i + 1], orr[4 * i + 2], orr[4 * i + 3]);
            }
          }
        } else {
          if (token < p.L)
            p.lse[batch_head * p.L + token] =
                fabsf(m_run) == INFINITY ? m_run : (m_run + log2f(l_run)) * 0.6931471805599453f;
          // into this block's Q tile, idle since its last S_q
          uint8_t* stage = q_tiles + ((live % QB) * N + q) * Q_TILE_BYTES;
#pragma unroll 1
          for (int h = 0; h < 2; ++h)
            stage_row64(o_tmem + h * 64, 1.f / l_run, limit <= 0, stage + h * Q_HALF_BYTES, row);
          fence_async_shared();
        }
        tc_fence_before();
        mbar_arrive(&st.o_read[q]);
      }
      if (nkv > 0) ++live;
      base += nkv;
      if (!ok || !advance(item)) break;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256 * N);
  }
}

// Joins the splits, one warp per query row: with m_i, l_i, O_i of split i and M = max m_i,
// O = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.  Splits where a row saw no key have l = 0 and an O that was never
// written; where it saw scores of -inf alone, m = -inf and l = NaN.  The splits are added in their order.
struct JoinParams {
  const float* part_o;
  const float2* part_ml;
  __nv_bfloat16* out;
  int64_t out_stride_b, out_stride_t;
  float* lse;
  int L, heads, splits;
  int64_t rows;  // batch * heads * L
};

__global__ void __launch_bounds__(256) attn_join_kernel(JoinParams p) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (row >= p.rows) return;
  const int64_t bh = row / p.L;
  const int token = static_cast<int>(row - bh * p.L);
  const int64_t first = bh * p.splits * p.L + token;
  float m = -INFINITY;
  for (int i = 0; i < p.splits; ++i) m = max_nan(m, p.part_ml[first + static_cast<int64_t>(i) * p.L].x);
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < p.splits; ++i) {
    const int64_t at = first + static_cast<int64_t>(i) * p.L;
    const float2 ml = p.part_ml[at];
    if (ml.y == 0.f || (ml.x == -INFINITY && m > ml.x)) continue;  // the same for the whole warp
    const float w = exp2f(ml.x - m);
    const float4 v = reinterpret_cast<const float4*>(p.part_o + at * HD)[lane];
    l = fmaf(w, ml.y, l);
    o.x = fmaf(w, v.x, o.x);
    o.y = fmaf(w, v.y, o.y);
    o.z = fmaf(w, v.z, o.z);
    o.w = fmaf(w, v.w, o.w);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t batch = bh / p.heads, head = bh - batch * p.heads;
  reinterpret_cast<uint2*>(p.out + batch * p.out_stride_b + token * p.out_stride_t + head * HD)[lane] =
      make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  if (lane == 0) p.lse[row] = fabsf(m) == INFINITY ? m : (m + log2f(l)) * 0.6931471805599453f;
}


}  // namespace attn
}  // namespace ogx
