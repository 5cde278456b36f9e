// Decode attention over the 8-bit paged KV cache (sm_100a): one query token per sequence.
//
//   s_j = scale * ks_{b(j)} (q . k8_j),   m = max_j s_j,   p_j = 2^(s_j - m),  l = sum_j p_j
//   o   = sum_j p_j vs_{b(j)} v8_j / l
//
// HBM-bound: every cache byte is used once per group of query heads, so the work is to keep
// enough bytes in flight on every SM and to spend few instructions per byte.
//
// Work split.  The keys of all (sequence, KV head) pairs form one line of 32-key tiles; each
// warp takes an equal, contiguous share of it (the sum over the lengths is repeated by every
// CTA, so no host length and no plan is needed).  Ragged batches, a single long sequence and
// many short ones all load the SMs evenly.  A pair that lies in one share is written at once; a
// pair cut by share boundaries leaves (m, l, O) partials that a second kernel joins in order, so
// results do not depend on timing.
//
// Each warp is its own pipeline: its lanes 0 and 1 issue the TMA loads of a tile's two 16-key
// slices (K and V, 128-byte-swizzled rows) STAGES tiles ahead and its 32 lanes consume them;
// no CTA barrier in the loop.
//
// Arithmetic.  The MMAs are transposed, S^T = K Q^T and O^T = V^T P^T, so that up to 8 query
// heads are the n = 8 columns: half the MMAs and registers of heads padded to 16 rows.  K codes
// come out of ldmatrix four dims per register and V codes, with the transposing 8-bit ldmatrix,
// four keys per register; the order of a contraction's index is free, so both feed the MMA after
// one cvt per pair, with q and the keys permuted to match.  K's second 8-key group starts at key
// 12 (then 13, 14, 15, 8 .. 11): both ldmatrix shapes then touch eight different swizzle rows.
// Weights are f16 (11 bits) scaled to 2^15 at most, which keeps those bits down to 2^-29 of the
// largest; vs enters through them relative to the largest vs so far.  m, l, O are fp32.
#include <ATen/Functions.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>

#include "attn_fp8.cuh"

namespace lb {
namespace fp8d {

using namespace fp8a;

constexpr int KT = 32;                        // keys per tile
constexpr int WARPS = 4;
constexpr int THREADS = 32 * WARPS;
constexpr int STAGES = 3;
constexpr int STAGE = 2 * 2 * SLICE;          // K slices, then V slices
constexpr int WARP_SMEM = STAGES * STAGE;
constexpr int MAX_SEQS = 4096;
constexpr float P_TOP = 32768.f;              // weights are p * 2^15

struct Work {
  float* part_o;      // [2 workers][heads of a chunk][D]
  float2* part_ml;    // [2 workers][heads of a chunk]
  int workers;        // warps of the grid
  int chunks;         // query-head chunks per KV head
};

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_t8(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float max_over_keys(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float sum_over_keys(float v) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Key (within a slice) of row r of the S^T tile.
__device__ __forceinline__ int key_of_row(int r) { return r < 8 ? r : 8 + ((r + 4) & 7); }

// First tile of each sequence (s_cum, in units of one tile of one head chunk) and its length.
// Every thread of the CTA takes part; the number of heads times chunks is `hc`.
__device__ void scan_lengths(const Args& a, int hc, int* s_cum, int* s_len, int* s_tot) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int base = 0;
  for (int b0 = 0; b0 < a.num_seqs; b0 += THREADS) {
    const int b = b0 + tid;
    int len = 0;
    if (b < a.num_seqs) {
      len = max(0, a.seq_lens[b]);
      const int64_t cap = static_cast<int64_t>(a.bt_width) << a.log2_bs;
      if (len > cap) {
        record_error(a.err, kErrBounds);
        len = static_cast<int>(cap);
      }
      s_len[b] = len;
    }
    int v = (len + KT - 1) / KT * hc;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    if (lane == 31) s_tot[warp] = v;
    __syncthreads();
    int all = 0;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) v += s_tot[w];
      all += s_tot[w];
    }
    if (b < a.num_seqs) s_cum[b + 1] = base + v;
    if (tid == 0 && b0 == 0) s_cum[0] = 0;
    base += all;
    __syncthreads();
  }
}

// Shares: worker w of n takes units [w U / n, (w + 1) U / n).  Fewer than two tiles a worker is
// not worth a partial result.
__device__ __forceinline__ int active_workers(int units, int workers) {
  return max(1, min(workers, units / 2));
}
__device__ __forceinline__ int share_begin(int w, int units, int n) {
  return static_cast<int>(static_cast<int64_t>(w) * units / n);
}
__device__ __forceinline__ int share_of(int unit, int units, int n) {
  return static_cast<int>(((static_cast<int64_t>(unit) + 1) * n - 1) / units);
}

// A position on the line of tiles.
struct Cursor {
  int b, h, t, nt;   // sequence, head chunk, tile, tiles of the sequence
  __device__ void seek(const int* cum, int n_seqs, int hc, int unit) {
    int lo = 0, hi = n_seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (cum[mid] <= unit) lo = mid;
      else hi = mid;
    }
    b = lo;
    nt = (cum[b + 1] - cum[b]) / hc;
    const int r = unit - cum[b];
    h = r / nt;
    t = r - h * nt;
  }
  // to the next tile; only called when one exists
  __device__ void next(const int* cum, int hc) {
    if (++t < nt) return;
    t = 0;
    if (++h < hc) return;
    h = 0;
    do {
      ++b;
      nt = cum[b + 1] - cum[b];
    } while (nt == 0);
    nt /= hc;
  }
};

template <int NT>   // query-head tiles of 8 per chunk
__global__ void __launch_bounds__(THREADS, 2)
    decode_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const Args a, const Work wk) {
  constexpr int HT = 8 * NT;                  // heads per chunk
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * WARP_SMEM;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + WARPS * WARP_SMEM) + warp * STAGES;
  // scales of a stage's slices: [stage][slice][ks, vs]
  float* s_scale = reinterpret_cast<float*>(smem + WARPS * WARP_SMEM + WARPS * STAGES * 8) +
                   warp * STAGES * 4;
  int* s_tot = reinterpret_cast<int*>(smem + WARPS * WARP_SMEM + WARPS * STAGES * 24);
  int* s_cum = s_tot + WARPS;
  int* s_len = s_cum + a.num_seqs + 1;
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(&full[s], 3);   // lane 0's expect + two scale loads
    fence_barrier_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  __syncwarp();
  pdl_trigger();
  pdl_wait();
  const int hc = a.hkv * wk.chunks;
  scan_lengths(a, hc, s_cum, s_len, s_tot);
  const int units = s_cum[a.num_seqs];
  if (units == 0) return;
  const int n_act = active_workers(units, wk.workers);
  const int w = warp * gridDim.x + blockIdx.x;   // neighbours on the line sit on different SMs
  if (w >= n_act) return;
  const int u_begin = share_begin(w, units, n_act), u_end = share_begin(w + 1, units, n_act);
  if (u_begin >= u_end) return;

  const int g = lane >> 2, t4 = lane & 3;
  const uint64_t pol = policy_evict_first();
  // ---- producer state: lanes 0 and 1 own the tile's slices; the block id of the next tile to
  // issue is fetched one tile early ----
  Cursor pc;
  pc.seek(s_cum, a.num_seqs, hc, u_begin);
  int pu = u_begin, p_id = 0;
  auto fetch_id = [&]() {
    const int key = pc.t * KT + lane * SL;
    if (lane < 2 && pu < u_end && key < s_len[pc.b])
      p_id = a.tables[pc.b * a.bt_stride + (key >> a.log2_bs)];
  };
  auto issue = [&](int stage) {
    if (pu >= u_end) return;                                       // warp-uniform
    const int key0 = pc.t * KT, len = s_len[pc.b];
    if (lane == 0)
      mbar_arrive_expect_tx(&full[stage], (len - key0 > SL ? 2 : 1) * 2 * SLICE);
    __syncwarp();
    if (lane < 2) {
      const int key = key0 + lane * SL;
      if (key < len) {
        const int blk = checked_block(a, p_id);
        const int bh = blk * a.hkv + pc.h / wk.chunks;
        const int row = (bh << a.log2_bs) + (key & ((1 << a.log2_bs) - 1));
        uint8_t* dst = ring + stage * STAGE + lane * SLICE;
        tma_load_2d(dst, &tmK, &full[stage], 0, row, pol);
        tma_load_2d(dst + 2 * SLICE, &tmV, &full[stage], 0, row, pol);
        const uint32_t sc = smem_u32(s_scale + stage * 4 + lane * 2);
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sc), "l"(a.k_scale + bh)
                     : "memory");
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(sc + 4), "l"(a.v_scale + bh)
                     : "memory");
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(
                       smem_u32(&full[stage]))
                   : "memory");
    }
    if (++pu < u_end) {
      pc.next(s_cum, hc);
      fetch_id();
    }
  };
  fetch_id();
#pragma unroll 1
  for (int s = 0; s < STAGES; ++s) issue(s);

  Cursor cc;
  cc.seek(s_cum, a.num_seqs, hc, u_begin);
  // row addresses of the two ldmatrix shapes
  const int krow = key_of_row(((lane >> 3) & 1) * 8 + (lane & 7));
  const int kchunk = lane >> 4;
  const int vi = lane & 15;
  const int vrow = key_of_row((vi >> 2) * 2 + (vi & 1) + ((vi & 2) ? 8 : 0));
  const uint32_t ring0 = smem_u32(ring);
  const uint32_t k_addr = ring0 + krow * D, v_addr = ring0 + 2 * SLICE + vrow * D;
  int stage = 0;
  uint32_t phase = 0;
  int u = u_begin, used = u_begin;               // used: tiles consumed, segment by segment u
  bool ok = true;
  while (u < u_end) {
    // ---- one (sequence, head chunk): tiles [t0, t1) ----
    const int t0 = cc.t, t1 = min(cc.nt, t0 + u_end - u), len = s_len[cc.b];
    const int kvh = cc.h / wk.chunks, head0 = kvh * a.group + (cc.h % wk.chunks) * HT;
    const int heads = min(HT, (kvh + 1) * a.group - head0);
    uint32_t qf[NT][8][2];
    float hs[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint2 raw[8];
      const bool have = n * 8 + g < heads;
      const bf16* qp = a.q + cc.b * a.q_ld + static_cast<int64_t>(head0 + n * 8 + g) * D + t4 * 4;
      float amax = 0.f;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        raw[c] = have ? *reinterpret_cast<const uint2*>(qp + c * 16) : make_uint2(0, 0);
        const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[c].x));
        const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[c].y));
        amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(y.x), fabsf(y.y)));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int sh = q_shift(amax);
      const float up = pow2i(sh);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[c].x));
        const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[c].y));
        qf[n][c][0] = pack_f16x2(x.x * up, x.y * up);
        qf[n][c][1] = pack_f16x2(y.x * up, y.y * up);
      }
      const float down = pow2i(-sh) * a.scale_log2;
      hs[n][0] = __shfl_sync(0xffffffffu, down, t4 * 8);
      hs[n][1] = __shfl_sync(0xffffffffu, down, t4 * 8 + 4);
    }
    float m[NT][2], l[NT][2], o[NT][8][4], vref = 7.5e-37f;   // 2^-120: below any useful scale
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[n][d][0] = o[n][d][1] = o[n][d][2] = o[n][d][3] = 0.f;
    }
    float inv_vref = P_TOP / vref;
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, nullptr));
      if (!ok) break;
      const int left = len - t * KT;                     // keys of this tile that exist
      const int nsl = left > SL ? 2 : 1;
      const float2 sc0 = *reinterpret_cast<const float2*>(s_scale + stage * 4);
      const float2 sc1 = nsl > 1 ? *reinterpret_cast<const float2*>(s_scale + stage * 4 + 2) : sc0;
      // ---- S^T = K Q^T ----
      float s[2][NT][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.f;
        if (i == 1 && nsl == 1) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
            s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = -INFINITY;
          break;
        }
        const uint32_t base = k_addr + stage * STAGE + i * SLICE;
#pragma unroll
        for (int c = 0; c < 8; c += 2) {
          uint32_t r[4], x[4], y[4];
          ldsm_x4(r, base + (((c + kchunk) ^ (krow & 7)) << 4));
          e4m3x4_to_f16(r[0], x[0], x[2]);
          e4m3x4_to_f16(r[1], x[1], x[3]);
          e4m3x4_to_f16(r[2], y[0], y[2]);
          e4m3x4_to_f16(r[3], y[1], y[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_f16(s[i][n], x[0], x[1], x[2], x[3], qf[n][c][0], qf[n][c][1]);
            mma_f16(s[i][n], y[0], y[1], y[2], y[3], qf[n][c + 1][0], qf[n][c + 1][1]);
          }
        }
        const float ks = i ? sc1.x : sc0.x;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          s[i][n][0] *= ks * hs[n][0];
          s[i][n][1] *= ks * hs[n][1];
          s[i][n][2] *= ks * hs[n][0];
          s[i][n][3] *= ks * hs[n][1];
        }
      }
      if (left < KT) {
        // keys past the end: whatever their memory holds, their score is -inf
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (i * SL + g >= left) s[i][n][0] = s[i][n][1] = -INFINITY;
            if (i * SL + key_of_row(8 + g) >= left) s[i][n][2] = s[i][n][3] = -INFINITY;
          }
      }
      // ---- running maximum and sum ----
      float corr[NT][2];
      bool moved = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = fmaxf(fmaxf(s[0][n][j], s[0][n][j + 2]), fmaxf(s[1][n][j], s[1][n][j + 2]));
          mx = fmaxf(m[n][j], max_over_keys(mx));
          const float safe = mx == -INFINITY ? 0.f : mx;
          corr[n][j] = ex2(m[n][j] - safe);
          moved |= mx != m[n][j];
          m[n][j] = mx;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            s[i][n][j] = ex2(s[i][n][j] - safe);
            s[i][n][j + 2] = ex2(s[i][n][j + 2] - safe);
          }
          l[n][j] = l[n][j] * corr[n][j] +
                    ((s[0][n][j] + s[0][n][j + 2]) + (s[1][n][j] + s[1][n][j + 2]));
        }
      const float vmax = fmaxf(sc0.y, sc1.y);
      float vcorr = 1.f;
      if (vmax > vref) {                                  // warp-uniform
        vcorr = vref / vmax;
        vref = vmax;
        inv_vref = P_TOP / vref;
      }
      if (__any_sync(0xffffffffu, moved || vcorr != 1.f)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float c0 = corr[n][0] * vcorr, c1 = corr[n][1] * vcorr;
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            o[n][d][0] *= c0;
            o[n][d][1] *= c1;
            o[n][d][2] *= c0;
            o[n][d][3] *= c1;
          }
        }
      }
      // ---- O^T += V^T P^T ----
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (i < nsl) {
          const float c = (i ? sc1.y : sc0.y) * inv_vref;
          uint32_t p[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            p[n][0] = transpose8(pack_f16x2(s[i][n][0] * c, s[i][n][1] * c));
            p[n][1] = transpose8(pack_f16x2(s[i][n][2] * c, s[i][n][3] * c));
          }
          // codes of keys past the end become zeros (NaN times weight 0 would be NaN)
          uint32_t keep = 0xffffffffu;
          if (left - i * SL < SL) {
            keep = 0;
#pragma unroll
            for (int y = 0; y < 4; ++y)
              if (key_of_row(2 * t4 + (y & 1) + (y & 2) * 4) < left - i * SL) keep |= 0xffu << (8 * y);
          }
          const uint32_t base = v_addr + stage * STAGE + i * SLICE;
#pragma unroll
          for (int c2 = 0; c2 < 8; c2 += 2) {
            uint32_t r[4], x[4];
            ldsm_t8(r, base + (((c2 + kchunk) ^ (vrow & 7)) << 4));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              e4m3x4_to_f16(r[2 * e] & keep, x[0], x[2]);
              e4m3x4_to_f16(r[2 * e + 1] & keep, x[1], x[3]);
#pragma unroll
              for (int n = 0; n < NT; ++n)
                mma_f16(o[n][c2 + e], x[0], x[1], x[2], x[3], p[n][0], p[n][1]);
            }
          }
        }
      }
      __syncwarp();      // every lane has read the stage: refill it
      issue(stage);
      ++used;
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (!ok) break;
    // ---- the pair's result, or this share's part of it ----
    const bool whole = t0 == 0 && t1 == cc.nt;
    const int slot = 2 * w + (t0 == 0 ? 1 : 0);
    const float vmul = vref * (1.f / P_TOP);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float l0 = sum_over_keys(l[n][0]), l1 = sum_over_keys(l[n][1]);
      const int h0 = n * 8 + 2 * t4;
      if (whole) {
        const float i0 = l0 != 0.f ? vmul / l0 : 0.f, i1 = l1 != 0.f ? vmul / l1 : 0.f;
        bf16* dst = a.out + cc.b * a.out_ld + static_cast<int64_t>(head0 + h0) * D + g;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          if (h0 < heads) {
            dst[d * 16] = __float2bfloat16(o[n][d][0] * i0);
            dst[d * 16 + 8] = __float2bfloat16(o[n][d][2] * i0);
          }
          if (h0 + 1 < heads) {
            dst[D + d * 16] = __float2bfloat16(o[n][d][1] * i1);
            dst[D + d * 16 + 8] = __float2bfloat16(o[n][d][3] * i1);
          }
        }
      } else {
        float* dst = wk.part_o + (static_cast<int64_t>(slot) * HT + h0) * D + g;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          dst[d * 16] = o[n][d][0] * vmul;
          dst[d * 16 + 8] = o[n][d][2] * vmul;
          dst[D + d * 16] = o[n][d][1] * vmul;
          dst[D + d * 16 + 8] = o[n][d][3] * vmul;
        }
        if (g == 0) {
          wk.part_ml[slot * HT + h0] = make_float2(m[n][0], l0);
          wk.part_ml[slot * HT + h0 + 1] = make_float2(m[n][1], l1);
        }
      }
    }
    u += t1 - t0;
    if (u < u_end) {
      cc.t = cc.nt - 1;
      cc.next(s_cum, hc);
    }
  }
  if (!ok) {
    // a load never arrived: report, and leave with none of this warp's copies in flight
    if (lane == 0) record_error(a.err, kErrTimeoutTmaFull);
    for (int i = 0; i < STAGES; ++i) {
      if (used + i < pu && !mbar_wait(&full[stage], phase, nullptr) && lane == 0)
        record_error(a.err, kErrTimeoutDrain);
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1u;
      }
    }
  }
}

// Joins the parts of the pairs that share boundaries cut, in the order of the keys; sequences
// without a key give 0.  One warp per (sequence, query head), 4 dims per lane.
template <int NT>
__global__ void __launch_bounds__(THREADS) join_kernel(const Args a, const Work wk) {
  constexpr int HT = 8 * NT;
  extern __shared__ int smem_i[];
  int* s_tot = smem_i;
  int* s_cum = s_tot + WARPS;
  int* s_len = s_cum + a.num_seqs + 1;
  pdl_trigger();
  pdl_wait();
  const int hc = a.hkv * wk.chunks;
  scan_lengths(a, hc, s_cum, s_len, s_tot);
  const int units = s_cum[a.num_seqs];
  const int n_act = active_workers(units, wk.workers);
  const int lane = threadIdx.x & 31;
  const int64_t rows = static_cast<int64_t>(a.num_seqs) * a.hq;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * WARPS + (threadIdx.x >> 5); i < rows;
       i += static_cast<int64_t>(gridDim.x) * WARPS) {
    const int b = static_cast<int>(i / a.hq), head = static_cast<int>(i % a.hq);
    const int nt = (s_cum[b + 1] - s_cum[b]) / hc;
    float o[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f, m = -INFINITY;
    if (nt > 0) {
      const int kvh = head / a.group, in = head % a.group;
      const int ua = s_cum[b] + (kvh * wk.chunks + in / HT) * nt, ub = ua + nt;
      const int wa = share_of(ua, units, n_act), wb = share_of(ub - 1, units, n_act);
      if (wa == wb) continue;                       // written whole by its warp
      const bool starts = share_begin(wa, units, n_act) <= ua;
      for (int w = wa; w <= wb; ++w) {
        const int64_t row = static_cast<int64_t>(2 * w + (w == wa && starts ? 1 : 0)) * HT + in % HT;
        const float2 ml = wk.part_ml[row];
        const float4 v = *reinterpret_cast<const float4*>(wk.part_o + row * D + lane * 4);
        const float mn = fmaxf(m, ml.x);
        const float safe = mn == -INFINITY ? 0.f : mn;
        const float c0 = ex2(m - safe), c1 = ex2(ml.x - safe);
        m = mn;
        l = l * c0 + ml.y * c1;
        o[0] = o[0] * c0 + v.x * c1;
        o[1] = o[1] * c0 + v.y * c1;
        o[2] = o[2] * c0 + v.z * c1;
        o[3] = o[3] * c0 + v.w * c1;
      }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    *reinterpret_cast<uint2*>(a.out + b * a.out_ld + static_cast<int64_t>(head) * D + lane * 4) =
        make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
  }
}

template <int NT>
void launch(const Args& a, const CUtensorMap& tk, const CUtensorMap& tv, const at::Tensor& like,
            cudaStream_t st) {
  constexpr int HT = 8 * NT;
  const size_t lens = (WARPS + 2 * static_cast<size_t>(a.num_seqs) + 1) * sizeof(int);
  const size_t smem = 1024 + WARPS * WARP_SMEM + WARPS * STAGES * 24 + lens;
  static bool attr = false;
  if (!attr) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(decode_kernel<NT>,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    attr = true;
  }
  Work wk;
  wk.chunks = (a.group + HT - 1) / HT;
  // two CTAs an SM while both fit (beyond about 2000 sequences the length tables leave room for
  // one); no more warps than tiles there can be
  const int per_sm = 2 * smem <= 226 * 1024 ? 2 : 1;
  const int64_t tiles = static_cast<int64_t>(a.num_seqs) * a.hkv * wk.chunks *
                        (((static_cast<int64_t>(a.bt_width) << a.log2_bs) + KT - 1) / KT);
  const int grid = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>(148 * per_sm, (tiles + 1) / 2)));
  wk.workers = grid * WARPS;
  at::Tensor ws = at::empty({static_cast<int64_t>(wk.workers) * 2 * HT * (D + 2)},
                            like.options().dtype(at::kFloat));
  wk.part_o = ws.data_ptr<float>();
  wk.part_ml = reinterpret_cast<float2*>(wk.part_o + static_cast<int64_t>(wk.workers) * 2 * HT * D);
  C10_CUDA_CHECK(launch_k(decode_kernel<NT>, dim3(grid), dim3(THREADS), smem, st, nullptr, 0, tk,
                          tv, a, wk));
  const int64_t rows = static_cast<int64_t>(a.num_seqs) * a.hq;
  C10_CUDA_CHECK(launch_k(join_kernel<NT>,
                          dim3(static_cast<int>(std::min<int64_t>((rows + WARPS - 1) / WARPS, 1184))),
                          dim3(THREADS), lens, st, nullptr, 0, a, wk));
}

}  // namespace fp8d

void fp8_decode(const fp8a::Args& a, const CUtensorMap& tk, const CUtensorMap& tv,
                const at::Tensor& like, cudaStream_t st) {
  TORCH_CHECK(a.num_seqs <= fp8d::MAX_SEQS, "paged_attention_fp8: at most ", fp8d::MAX_SEQS,
              " sequences");
  TORCH_CHECK(static_cast<int64_t>(a.num_seqs) * a.hq *
                      ((static_cast<int64_t>(a.bt_width) << a.log2_bs) / fp8d::KT + 1) <
                  (int64_t(1) << 31),
              "paged_attention_fp8: sequences x heads x table width too large");
  if (a.group <= 8) fp8d::launch<1>(a, tk, tv, like, st);
  else fp8d::launch<2>(a, tk, tv, like, st);
}

}  // namespace lb
