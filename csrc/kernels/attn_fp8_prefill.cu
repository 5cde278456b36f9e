// Prefill / verify attention over the 8-bit paged KV cache on tcgen05 (sm_100a).
//
//   s_j = scale * ks_{b(j)} (q . k8_j),   o = sum_j 2^(s_j - m) vs_{b(j)} v8_j / sum_j 2^(s_j - m)
//
// One CTA = 256 packed query rows (token, head in group) of one sequence x one KV head, as two
// 128-row tiles that alternate on the tensor core; keys in tiles of 128.  Compute-bound: 4 * 128
// FLOP per (row, key) against one exponential each, so the tensor core and the softmax have to
// overlap, and everything else must stay out of their way:
//
//   warp 0      TMA: the 8-bit K and V tiles, 16-key slices, lane i slice i, into two staging
//               buffers (K, V, K, V, ...).
//   warp 1      MMA issuer and TMEM owner.  The two query tiles share one S region: a tile's softmax
//               holds S in registers soon after it is written, and the region goes to the other tile.
//               With slots (tile 0, 0), (tile 1, 0), (tile 0, 1), ... the issue order is S(s),
//               O += P(s - 2) V: a softmax that ends finds its next S written, its P V runs under it,
//               and the two softmax groups settle half a period apart, one in its exponentials while
//               the other loads and compares.  P has columns of its own, so no MMA writes what
//               another (of another shape, whose order is not defined) may still read.
//   warp 2      the slices' scales of a tile, four tiles ahead.
//   warps 4-7   convert staged codes to f16 tiles in the MMA's swizzled layout.  The codes go in
//               unscaled: e4m3 is exact in f16, so the conversion is one cvt per pair, and rows past
//               the sequence's end become zeros.
//   warps 8-15  softmax, one thread per query row: it reads its row of q once (as f16, scaled by a
//               power of two and with the softmax scale's sign, into shared memory), then per tile 128
//               scores from TMEM.  ks of a 16-key slice multiplies its scores, vs goes into the exponent:
//                 P = 2^(s + log2 vs - m' + 7),  m' >= max(s + log2 vs) - 8,
//               so P is at most 2^15 and keeps f16's 11 bits down to 2^-21 of the largest contribution;
//               l sums P / vs in fp32 (a scale of 0 stands for a block of zeros: any other does too).  m'
//               moves only when the maximum passes it by 2^8 (then O is rescaled in TMEM, after the
//               previous tile's P V).
// P (f16, in TMEM) is the MMA's A operand; V is read in its key-major layout.  TMEM: O_t at 128 t, S at
// 256, P_t at 384 + 64 t.  Registers: 512 threads start with 128 each; the softmax warps take 200
// (40 + 72 + 200 + 200 = 4 * 128 per quarter).  Every wait is bounded; on expiry the kernel records an
// error and unwinds.
//
// Measured (32 / 8 heads): 2 x 512 tokens over 4k 86 us (750 TFLOP/s, 44 % of the measured bf16 burst),
// 2048 tokens over 18k 657 us (889 TFLOP/s, 53 %); on the fastest box met 78 and 595, where the
// variants below were timed.  The MMAs alone take 448 us of the latter; the softmax warps bind it (about
// 2400 cycles of a tile's 4000 go to the exponentials and their conversion, of which the 128 exponentials
// themselves need 1024).  Tried: an S region per tile with P written over it 701 us; units of 64 keys with
// two S regions 734 us; every fourth pair of exponentials as a cubic on the FMA pipe 689 us.  Where the
// compiler places the loop moves the time by up to 10 % (634 to 707 us for changes outside it).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>

#include "attn_fp8.cuh"

namespace lb {
namespace fp8p {

using namespace fp8a;

constexpr int QT = 2;
constexpr int BM = 128 * QT;
constexpr int BN = 128;                   // keys per tile
constexpr int NSL = BN / SL;              // slices per tile
constexpr int THREADS = 512;
constexpr int HALF = BN * 128;            // f16 tile: two 64-dim halves of 128-byte rows
constexpr int TILE = 2 * HALF;
constexpr int STAGED = BN * D;            // 8-bit tile
constexpr int KST = 2, VST = 2, SST = 2, CST = 4;
constexpr int SMEM_Q = 0;
constexpr int SMEM_K = QT * TILE;
constexpr int SMEM_V = SMEM_K + KST * TILE;
constexpr int SMEM_S = SMEM_V + VST * TILE;
constexpr int SMEM_C = SMEM_S + SST * STAGED;          // [CST][NSL] float4 slice constants
constexpr int SMEM_BAR = SMEM_C + CST * NSL * 16;
constexpr int SMEM_TOTAL = SMEM_BAR + 256 + 1024;
constexpr uint32_t TMEM_COLS = 512;
constexpr float LAZY = 8.f, SHIFT = 7.f;
// Added to the factor of the raw scores (at most 2^31 of them in size), so that it is never zero: a masked
// score is -inf, and -inf * 0 would be NaN.  Moves a score by less than 2^-94.
constexpr float TINY = 1.17549435e-38f;   // 2^-126

__device__ __forceinline__ uint64_t sw128_mnmajor_desc(uint32_t saddr, uint32_t lbo_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((lbo_bytes >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}
// kind::f16 with f16 A and B, fp32 D.
constexpr uint32_t idesc_f16(int M, int N, int b_mn_major) {
  return (1u << 4) | (static_cast<uint32_t>(b_mn_major) << 16) |
         (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}
// One lane of a converged warp.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r;
}
// MMAs and commits of the elected lane of a converged warp (the forms of common.cuh are for code
// that a single lane runs).
__device__ __forceinline__ void mma_ss_if(uint32_t leader, uint32_t d_tmem, uint64_t a_desc,
                                          uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts_if(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem,
                                          uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          smem_u32(bar)),
      "r"(leader)
      : "memory");
}
__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void regs_take() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_give() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ uint64_t pack_f2(float lo, float hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__global__ void __launch_bounds__(THREADS, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  auto sQ = [&](int t) { return smem + SMEM_Q + t * TILE; };
  auto sK = [&](int s) { return smem + SMEM_K + s * TILE; };
  auto sV = [&](int s) { return smem + SMEM_V + s * TILE; };
  auto sS = [&](int s) { return smem + SMEM_S + s * STAGED; };
  float4* sC = reinterpret_cast<float4*>(smem + SMEM_C);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + SMEM_BAR);
  uint64_t* q_full = bars;                 // Q of both tiles in shared memory (8 softmax warps)
  uint64_t* st_full = q_full + 1;          // [SST] staged codes (TMA)
  uint64_t* st_empty = st_full + SST;      // [SST] read by the 4 converter warps
  uint64_t* k_full = st_empty + SST;       // [KST] f16 tile written (4 converter warps)
  uint64_t* k_empty = k_full + KST;        // [KST] S of every query tile done
  uint64_t* v_full = k_empty + KST;        // [VST]
  uint64_t* v_empty = v_full + VST;        // [VST] P V of every query tile done
  uint64_t* c_full = v_empty + VST;        // [CST] slice constants
  uint64_t* c_empty = c_full + CST;        // [CST] read by the 8 softmax warps
  uint64_t* s_full = c_empty + CST;        // [QT] S of a tile's slot (and all earlier MMAs)
  uint64_t* s_free = s_full + QT;          // S of a slot in registers (4 softmax warps)
  uint64_t* p_ready = s_free + 1;          // [QT] P_t in TMEM (4 softmax warps)
  uint64_t* pv_done = p_ready + QT;        // [QT] P_t V
  uint64_t* mma_drain = pv_done + QT;      // every MMA issued, after an abort
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int kvh = blockIdx.y;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 8);
    for (int s = 0; s < SST; ++s) {
      mbar_init(&st_full[s], 1);
      mbar_init(&st_empty[s], 4);
    }
    for (int s = 0; s < KST; ++s) {
      mbar_init(&k_full[s], 4);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < VST; ++s) {
      mbar_init(&v_full[s], 4);
      mbar_init(&v_empty[s], 1);
    }
    for (int s = 0; s < CST; ++s) {
      mbar_init(&c_full[s], 1);
      mbar_init(&c_empty[s], 8);
    }
    mbar_init(s_free, 4);
    mbar_init(mma_drain, 1);
    for (int t = 0; t < QT; ++t) {
      mbar_init(&s_full[t], 1);
      mbar_init(&p_ready[t], 4);
      mbar_init(&pv_done[t], 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  pdl_trigger();
  pdl_wait();

  const int seq = a.tile_seq[blockIdx.x];
  const int item_row0 = a.tile_row0[blockIdx.x];
  const bool bad = seq >= a.num_seqs || item_row0 < 0;
  const bool used = seq >= 0 && !bad;
  if (bad && threadIdx.x == 0) record_error(a.err, kErrBounds);
  const int q_start = used ? a.cu_q[seq] : 0;
  int q_len = used ? a.cu_q[seq + 1] - q_start : 0;
  if (q_start < 0 || q_len < 0 || q_len > a.tokens - q_start) {
    if (threadIdx.x == 0) record_error(a.err, kErrBounds);
    q_len = 0;
  }
  int kv_len = used ? max(0, a.seq_lens[seq]) : 0;
  const int64_t cap = static_cast<int64_t>(a.bt_width) << a.log2_bs;
  if (kv_len > cap) {
    if (threadIdx.x == 0) record_error(a.err, kErrBounds);
    kv_len = static_cast<int>(cap);
  }
  const int nrows_seq = q_len * a.group;
  // an item past the sequence's rows has none; row0 + BM below must not pass 2^31
  const int row0 = min(item_row0, nrows_seq);
  const int nqt = row0 + 128 < nrows_seq ? QT : 1;
  const int* btab = a.tables + (used ? seq * a.bt_stride : 0);
  // keys this CTA needs: causal rows see keys <= kv_len - q_len + token
  int k_limit = row0 < nrows_seq ? kv_len : 0;
  if (a.causal && k_limit > 0) {
    const int last_row = min(row0 + BM, nrows_seq) - 1;
    k_limit = min(kv_len, kv_len - q_len + last_row / a.group + 1);
  }
  const int ntiles = k_limit > 0 ? (k_limit + BN - 1) / BN : 0;
  const int bs_mask = (1 << a.log2_bs) - 1;

  int st_par[SST] = {-1, -1};    // producer: parity of the last load issued per buffer
  if (warp < 4) {
    regs_give<40>();
    if (warp == 0 && ntiles > 0) {
      // lane i < NSL owns slice i; its block id is fetched one tile early
      const uint64_t pol = policy_evict_last();
      auto slice_id = [&](int j) {
        const int key = j * BN + lane * SL;
        return lane < NSL && key < kv_len ? btab[key >> a.log2_bs] : 0;
      };
      int id = slice_id(0);
      bool ok = true;
      for (int j = 0; j < ntiles && ok; ++j) {
        const int next = j + 1 < ntiles ? slice_id(j + 1) : 0;
        const int key = j * BN + lane * SL;
        const int n = min(NSL, (kv_len - j * BN + SL - 1) / SL);
        const int blk = lane < n ? checked_block(a, id) : 0;
        const int row = ((blk * a.hkv + kvh) << a.log2_bs) + (key & bs_mask);
        for (int kv = 0; kv < 2 && ok; ++kv) {
          const int i = 2 * j + kv, s = i % SST;
          ok = __all_sync(0xffffffffu, mbar_wait(&st_empty[s], ((i / SST) & 1) ^ 1u, abort_flag));
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&st_full[s], n * SLICE);
          __syncwarp();
          if (lane < n)
            tma_load_2d(sS(s) + lane * SLICE, kv ? &tmV : &tmK, &st_full[s], 0, row, pol);
          st_par[s] = (i / SST) & 1;
        }
        id = next;
      }
      if (!ok) {
        if (lane == 0) record_error(a.err, kErrTimeoutSmemEmpty);
        *abort_flag = 1;
      }
    } else if (warp == 1 && ntiles > 0) {
      constexpr uint32_t idesc_s = idesc_f16(128, BN, 0);
      constexpr uint32_t idesc_o = idesc_f16(128, D, 1);
      const uint32_t colS = tmem_base + 256;
      static_assert(KST == 2 && VST == 2, "parities below");
      const uint32_t leader = elect_one();
      const uint64_t q_desc = sw128_kmajor_desc(smem_u32(sQ(0)));
      const uint64_t k_desc = sw128_kmajor_desc(smem_u32(sK(0)));
      const uint64_t v_desc = sw128_mnmajor_desc(smem_u32(sV(0)), HALF);
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0;
      };
      auto issue_s = [&](int s) {
        const int t = nqt == 2 ? s & 1 : 0, j = nqt == 2 ? s >> 1 : s;
        if (t == 0 && !wait(&k_full[j & 1], (j >> 1) & 1)) return false;
        if (s > 0 && !wait(s_free, (s - 1) & 1)) return false;
        tc_fence_after();
        const uint64_t qd = q_desc + ((t * TILE) >> 4), kd = k_desc + (((j & 1) * TILE) >> 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = ((k >> 2) * HALF + (k & 3) * 32) >> 4;
          mma_ss_if(leader, colS, qd + off, kd + off, idesc_s, k > 0 ? 1u : 0u);
        }
        commit_if(leader, &s_full[t]);   // arrives once this and every earlier MMA are done
        if (t == nqt - 1) commit_if(leader, &k_empty[j & 1]);
        return true;
      };
      auto issue_pv = [&](int s) {
        const int t = nqt == 2 ? s & 1 : 0, j = nqt == 2 ? s >> 1 : s;
        if (t == 0 && !wait(&v_full[j & 1], (j >> 1) & 1)) return false;
        if (!wait(&p_ready[t], j & 1)) return false;
        tc_fence_after();
        const uint64_t vd = v_desc + (((j & 1) * TILE) >> 4);
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)
          mma_ts_if(leader, tmem_base + 128 * t, tmem_base + 384 + 64 * t + k * 8,
                    vd + ((k * 16 * 128) >> 4), idesc_o, (j > 0 || k > 0) ? 1u : 0u);
        if (t == nqt - 1) commit_if(leader, &v_empty[j & 1]);
        commit_if(leader, &pv_done[t]);
        return true;
      };
      const int slots = nqt * ntiles;
      bool ok = wait(q_full, 0);
      for (int s = 0; ok && s < slots; ++s) {
        ok = issue_s(s);
        if (ok && s >= nqt) ok = issue_pv(s - nqt);
      }
      for (int s = slots - nqt; ok && s < slots; ++s) ok = issue_pv(s);
      if (!ok) {
        if (lane == 0) record_error(a.err, kErrTimeoutTmaFull);
        *abort_flag = 1;
      }
    } else if (warp == 2 && ntiles > 0) {
      // slice constants, vs relative to the first slice's vs0: ks, log2(vs / vs0), vs0 / vs, vs0
      auto slice_id = [&](int j) {
        const int key = j * BN + lane * SL;
        return lane < NSL && key < kv_len ? btab[key >> a.log2_bs] : -1;
      };
      int id = slice_id(0);
      float lv0 = 0.f, vs0 = 1.f;
      for (int j = 0; j < ntiles; ++j) {
        const int next = j + 1 < ntiles ? slice_id(j + 1) : -1;
        float ks = 0.f, vs = 0.f;
        const bool have = lane < NSL && j * BN + lane * SL < kv_len;
        if (have) {
          const int64_t bh = static_cast<int64_t>(checked_block(a, id)) * a.hkv + kvh;
          ks = a.k_scale[bh];
          vs = a.v_scale[bh];
        }
        if (vs == 0.f) vs = vs0;     // a block of zeros: any positive scale stands for it
        const float lv = log2f(vs);
        if (j == 0) {
          lv0 = __shfl_sync(0xffffffffu, lv, 0);
          vs0 = __shfl_sync(0xffffffffu, vs, 0);
        }
        if (!__all_sync(0xffffffffu, mbar_wait(&c_empty[j % CST], ((j / CST) & 1) ^ 1u, abort_flag))) {
          if (lane == 0) record_error(a.err, kErrTimeoutSmemEmpty);
          *abort_flag = 1;
          break;
        }
        // slices past the end hold masked scores only
        if (lane < NSL)
          sC[(j % CST) * NSL + lane] =
              have ? make_float4(ks, lv - lv0, exp2f(lv0 - lv), vs0) : make_float4(1.f, 0.f, 0.f, vs0);
        __syncwarp();
        if (lane == 0) mbar_arrive(&c_full[j % CST]);
        id = next;
      }
    }
  } else if (warp < 8) {
    regs_give<72>();
    // ---- converters: thread handles 16-byte pieces (16 codes) of the staged rows ----
    const int ct = threadIdx.x - 128;
    const int c = ct & 7;                       // 16-dim chunk of the row
    const int half = c >> 2;
    bool ok = true;
    for (int i = 0; i < 2 * ntiles && ok; ++i) {
      const int j = i >> 1, kv = i & 1, s = i % SST;
      uint64_t* dst_full = kv ? &v_full[j % VST] : &k_full[j % KST];
      uint64_t* dst_empty = kv ? &v_empty[j % VST] : &k_empty[j % KST];
      const uint32_t par = ((j / (kv ? VST : KST)) & 1);
      ok = __all_sync(0xffffffffu, mbar_wait(&st_full[s], (i / SST) & 1, abort_flag)) &&
           __all_sync(0xffffffffu, mbar_wait(dst_empty, par ^ 1u, abort_flag));
      if (!ok) break;
      const uint8_t* src = sS(s);
      uint8_t* dst = (kv ? sV(j % VST) : sK(j % KST)) + half * HALF;
      uint4 raw[BN / 16];
#pragma unroll
      for (int r = 0; r < BN / 16; ++r)
        raw[r] = *reinterpret_cast<const uint4*>(src + (r * 16 + (ct >> 3)) * D +
                                                 ((c ^ ((ct >> 3) & 7)) << 4));
#pragma unroll
      for (int r = 0; r < BN / 16; ++r) {
        const int row = r * 16 + (ct >> 3);
        const bool live = j * BN + row < kv_len;
        uint32_t f[8];
        e4m3x4_to_f16(live ? raw[r].x : 0u, f[0], f[1]);
        e4m3x4_to_f16(live ? raw[r].y : 0u, f[2], f[3]);
        e4m3x4_to_f16(live ? raw[r].z : 0u, f[4], f[5]);
        e4m3x4_to_f16(live ? raw[r].w : 0u, f[6], f[7]);
        // the second half's threads store their pieces in the other order: eight threads then
        // touch eight different 16-byte banks
        const int first = 2 * (c & 3) + half;
        const uint4 lo = make_uint4(f[0], f[1], f[2], f[3]), hi = make_uint4(f[4], f[5], f[6], f[7]);
        *reinterpret_cast<uint4*>(dst + row * 128 + ((first ^ (row & 7)) << 4)) = half ? hi : lo;
        *reinterpret_cast<uint4*>(dst + row * 128 + (((first ^ 1) ^ (row & 7)) << 4)) = half ? lo : hi;
      }
      // The staging buffer is given back only here, when every loaded code has been used: an arrival
      // placed right behind the loads let TMA's next tile overtake some of them.
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&st_empty[s]);
        mbar_arrive(dst_full);
      }
    }
    if (!ok) {
      if (lane == 0) record_error(a.err, kErrTimeoutTmaFull);
      *abort_flag = 1;
    }
  } else {
    regs_take<200>();
    // ---- softmax / epilogue: warpgroup t = query tile t, thread = query row (TMEM lane) ----
    const int t = (warp - 8) >> 2;
    const int quad = warp & 3;
    const int r = quad * 32 + lane;
    const int pr = row0 + 128 * t + r;
    const bool valid_row = pr < nrows_seq;
    const int tok = valid_row ? pr / a.group : 0;
    const int head = kvh * a.group + (valid_row ? pr - tok * a.group : 0);
    const int qpos = kv_len - q_len + tok;
    const int klim = !valid_row ? 0 : (a.causal ? min(kv_len, qpos + 1) : kv_len);
    float row_scale = 0.f;
    if (t < nqt && ntiles > 0) {
      uint4 raw[16];
      const uint4* src = reinterpret_cast<const uint4*>(
          a.q + static_cast<int64_t>(q_start + tok) * a.q_ld + static_cast<int64_t>(head) * D);
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        raw[i] = valid_row ? src[i] : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
          amax = fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y)));
        }
      }
      const int sh = q_shift(amax);
      // a negative softmax scale turns q's sign: row_scale stays positive, so the maximum of a slice's
      // raw scores is that of its scaled ones
      const float up = copysignf(pow2i(sh), a.scale_log2);
      row_scale = pow2i(-sh) * fabsf(a.scale_log2);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
          h[k] = pack_f16x2(x.x * up, x.y * up);
        }
        *reinterpret_cast<uint4*>(sQ(t) + (i >> 3) * HALF + r * 128 + (((i & 7) ^ (r & 7)) << 4)) =
            make_uint4(h[0], h[1], h[2], h[3]);
      }
      fence_async_smem();
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);

    const uint32_t tl = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t colO = 128 * t, colS = 256, colP = 384 + 64 * t;
    float m_used = -INFINITY, l = 0.f, vs0 = 0.f;
    bool ok = true;
    if (t >= nqt) {
      // no rows in this tile: only take part in the constants' ring
      for (int j = 0; j < ntiles && ok; ++j) {
        ok = __all_sync(0xffffffffu, mbar_wait(&c_full[j % CST], (j / CST) & 1, abort_flag));
        if (ok && lane == 0) mbar_arrive(&c_empty[j % CST]);
      }
    }
    // tiles that every row of the warp sees whole need no mask
    const int clear = __reduce_min_sync(0xffffffffu, klim) / BN;
    for (int j = 0; j < ntiles && t < nqt; ++j) {
      ok = __all_sync(0xffffffffu, mbar_wait(&c_full[j % CST], (j / CST) & 1, abort_flag) &&
                                       mbar_wait(&s_full[t], j & 1, abort_flag));
      if (!ok) break;
      tc_fence_after();
      uint32_t sr[BN];
#pragma unroll
      for (int c = 0; c < 4; ++c)
        tmem_ld32(tl + colS + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(sr + 32 * c));
      float sc[NSL], lv[NSL];
      const float4* cst = sC + (j % CST) * NSL;
#pragma unroll
      for (int i = 0; i < NSL; ++i) {
        const float4 v = cst[i];
        sc[i] = fmaf(v.x, row_scale, TINY);
        lv[i] = v.y;
        vs0 = v.w;
      }
      tc_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(s_free);
      if (j >= clear) {
        const int nvalid = min(BN, max(0, klim - j * BN));
#pragma unroll
        for (int c = 0; c < BN; ++c)
          if (c >= nvalid) sr[c] = __float_as_uint(-INFINITY);
      }
      // ks > 0 keeps a slice's order: maximum of the raw scores first, then its scale
      float mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < NSL; ++i) {
        float x = __uint_as_float(sr[16 * i]), y = __uint_as_float(sr[16 * i + 1]);
#pragma unroll
        for (int c = 2; c < 16; c += 4) {
          x = max3f(x, __uint_as_float(sr[16 * i + c]), __uint_as_float(sr[16 * i + c + 1]));
          if (c + 2 < 16)
            y = max3f(y, __uint_as_float(sr[16 * i + c + 2]), __uint_as_float(sr[16 * i + c + 3]));
        }
        mx = fmaxf(mx, fmaf(fmaxf(x, y), sc[i], lv[i]));
      }
      // the previous P V has read P and is in O (it was issued when that P was ready, a softmax ago)
      if (j > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[t], (j - 1) & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
      }
      const bool need = mx > m_used + LAZY;
      if (__any_sync(0xffffffffu, need)) {
        const float m_new = need ? mx : m_used;
        const float corr = need ? ex2(m_used - m_new) : 1.f;
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t ov[32];
            tmem_ld32(tl + colO + 32 * c, ov);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * corr);
            tmem_st16(tl + colO + 32 * c, *reinterpret_cast<uint32_t(*)[16]>(ov));
            tmem_st16(tl + colO + 32 * c + 16, *reinterpret_cast<uint32_t(*)[16]>(ov + 16));
          }
        }
        l *= corr;
        m_used = m_new;
      }
      const float ms = SHIFT - (m_used == -INFINITY ? 0.f : m_used);
      // exponents first, in place: the exponentials then follow each other without waiting
#pragma unroll
      for (int i = 0; i < NSL; ++i) {
        const float add = lv[i] + ms;
        const uint64_t sc2 = pack_f2(sc[i], sc[i]), ad2 = pack_f2(add, add);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const int e = 16 * i + 2 * c;
          float x0, x1;
          unpack_f2(fma_f2(pack_f2(__uint_as_float(sr[e]), __uint_as_float(sr[e + 1])), sc2, ad2),
                    x0, x1);
          sr[e] = __float_as_uint(x0);
          sr[e + 1] = __float_as_uint(x1);
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t pk[16];
#pragma unroll
        for (int c = 0; c < 32; ++c) sr[32 * q + c] = __float_as_uint(ex2(__uint_as_float(sr[32 * q + c])));
#pragma unroll
        for (int c = 0; c < 16; ++c)
          pk[c] = pack_f16x2(__uint_as_float(sr[32 * q + 2 * c]), __uint_as_float(sr[32 * q + 2 * c + 1]));
        tmem_st16(tl + colP + 16 * q, pk);
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
          const uint32_t* p = sr + 32 * q + 16 * i2;
          uint64_t t4[4];
#pragma unroll
          for (int c = 0; c < 4; ++c)
            t4[c] = add_f2(pack_f2(__uint_as_float(p[4 * c]), __uint_as_float(p[4 * c + 1])),
                           pack_f2(__uint_as_float(p[4 * c + 2]), __uint_as_float(p[4 * c + 3])));
          float la, lb;
          unpack_f2(add_f2(add_f2(t4[0], t4[1]), add_f2(t4[2], t4[3])), la, lb);
          l = fmaf(la + lb, cst[2 * q + i2].z, l);
        }
      }
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&p_ready[t]);
        mbar_arrive(&c_empty[j % CST]);
      }
    }
    if (!ok) {
      if (lane == 0) record_error(a.err, kErrTimeoutTmemFull);
      *abort_flag = 1;
    }
    // ---- epilogue: O_t / l -> out[token][head][:]; rows that saw no key give 0 ----
    if (ok && t < nqt && ntiles > 0) {
      ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[t], (ntiles - 1) & 1, abort_flag));
      if (!ok) {
        if (lane == 0) record_error(a.err, kErrTimeoutTmemFull);
        *abort_flag = 1;
      }
      tc_fence_after();
    }
    if (ok && t < nqt) {
      const float inv = l != 0.f ? 1.f / l : 0.f;
      bf16* dst = a.out + static_cast<int64_t>(q_start + tok) * a.out_ld +
                  static_cast<int64_t>(head) * D;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t ov[32];
        if (ntiles > 0) {                       // uniform
          tmem_ld32(tl + colO + 32 * c, ov);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = 0;
        }
        if (valid_row) {
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * inv * vs0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint4 v;
            v.x = pack_bf16x2(__uint_as_float(ov[8 * i]), __uint_as_float(ov[8 * i + 1]));
            v.y = pack_bf16x2(__uint_as_float(ov[8 * i + 2]), __uint_as_float(ov[8 * i + 3]));
            v.z = pack_bf16x2(__uint_as_float(ov[8 * i + 4]), __uint_as_float(ov[8 * i + 5]));
            v.w = pack_bf16x2(__uint_as_float(ov[8 * i + 6]), __uint_as_float(ov[8 * i + 7]));
            *reinterpret_cast<uint4*>(dst + 32 * c + 8 * i) = v;
          }
        }
      }
    }
  }

  // after an abort: wait (bounded) for this CTA's MMAs and TMA copies still in flight
  __syncthreads();
  if (warp == 1 && *abort_flag) {
    commit_if(elect_one(), mma_drain);         // of the lane that issued the MMAs
    if (!mbar_wait(mma_drain, 0, nullptr) && lane == 0) record_error(a.err, kErrTimeoutDrain);
  }
  if (warp == 0 && lane == 0 && *abort_flag) {
    bool drained = true;
    for (int s = 0; s < SST; ++s)
      if (st_par[s] >= 0)
        drained &= mbar_wait(&st_full[s], static_cast<uint32_t>(st_par[s]), nullptr, kWaitBudgetNs);
    if (!drained) record_error(a.err, kErrTimeoutDrain);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

}  // namespace fp8p

void fp8_prefill(const fp8a::Args& a, const CUtensorMap& tk, const CUtensorMap& tv,
                 cudaStream_t st) {
  using namespace fp8p;
  static std::atomic<bool> allowed[64] = {};
  allow_smem(prefill_kernel, SMEM_TOTAL, allowed);
  C10_CUDA_CHECK(launch_k(prefill_kernel, dim3(a.num_tiles, a.hkv), dim3(THREADS), SMEM_TOTAL, st,
                          nullptr, 0, tk, tv, a));
}

}  // namespace lb
