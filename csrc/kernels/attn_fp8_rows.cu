// Attention over the 8-bit paged KV cache for few query rows per sequence (sm_100a): decode (one
// token) and short chunks such as speculative verification.
//
//   t_j = log2(e) scale * ks_{b(j)} (q . k8_j) + log2 vs_{b(j)},   m = max_j t_j,   w_j = 2^(t_j - m)
//   o   = sum_j w_j v8_j / sum_j w_j / vs_{b(j)}
//
// HBM-bound: every cache byte is used once per few query rows, so the work is to keep enough bytes
// in flight on every SM and to spend few instructions per byte.
//
// Work split.  An entry is a sequence (decode) or an item of the work list; its query rows (token,
// head in group) are cut into chunks of 8, 16 or 24 columns, and (KV head, chunk) over the entry's keys
// is a run of 32-key tiles.  All runs form one line; each warp takes an equal, contiguous share of
// it (the sum over the lengths is repeated by every CTA, so no host length and no plan is needed).
// Ragged batches, a single long sequence and many short ones all load the SMs evenly.  A run that
// lies in one share is written at once; a run cut by share boundaries leaves (m, l, O) partials that
// a second kernel joins in order, so results do not depend on timing.
//
// Each warp is its own pipeline: its lanes 0 and 1 issue the TMA loads of a tile's two 16-key
// slices (K and V, 128-byte-swizzled rows) STAGES tiles ahead and its 32 lanes consume them;
// no CTA barrier in the loop.
//
// Arithmetic.  The MMAs are transposed, S^T = K Q^T and O^T = V^T P^T, so that up to 8 query
// rows are the n = 8 columns: half the MMAs and registers of rows padded to 16.  K codes
// come out of ldmatrix four dims per register and V codes, with the transposing 8-bit ldmatrix,
// four keys per register; the order of a contraction's index is free, so both feed the MMA after
// one cvt per pair, with q and the keys permuted to match.  K's second 8-key group starts at key
// 12 (then 13, 14, 15, 8 .. 11): both ldmatrix shapes then touch eight different swizzle rows.
// Weights are f16 (11 bits) scaled to 2^15 at most, which keeps those bits down to 2^-29 of the
// largest.  vs is part of a weight's exponent, so a block counts by its softmax weight times its scale,
// however far its scale lies from the others'.  l sums w / vs relative to the share's first vs (not scaled
// by 2^15), so vs may spread over 2^100 in a sequence and head.  A scale of 0 stands for a block of zeros: its
// keys count in l with the first vs's exponent.  m, l, O are fp32.
//
// Measured (32 query / 8 KV heads unless said): 256 ragged sequences up to 2304 keys 117 us (5.5 TB/s,
// 84 % of the measured copy rate; the main kernel alone 108 us), 37 x 3001 with 32 KV heads 84 us (87 %),
// 7 sequences up to 100k keys with 64 / 8 heads 132 us (87 %), one of 2047 keys 9.8 us (launches and
// the first loads), 32 x up to 5 tokens over up to 1280 keys 28 us.  With 8 warps an SM instead of 12
// the first took 126 us: two warps a scheduler leave it idle most of the time.
#include <ATen/Functions.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>

#include <type_traits>

#include "attn_fp8.cuh"

namespace lb {
namespace fp8d {

using namespace fp8a;

constexpr int KT = 32;                        // keys per tile
constexpr int WARPS = 4;
constexpr int THREADS = 32 * WARPS;
constexpr int STAGE = 2 * 2 * SLICE;          // K slices, then V slices
// One column tile of 8: 2 stages and 12 warps an SM; two: 3 stages and 8 warps (their O takes twice
// the registers): 192 KB of an SM in flight.  Three: 2 stages, and q's fragments wait in shared
// memory, each lane's own, instead of 48 registers.
constexpr int stages_of(int nt) { return nt == 2 ? 3 : 2; }
constexpr int ctas_of(int nt) { return nt == 1 ? 3 : 2; }
constexpr int q_smem_of(int nt) { return nt > 2 ? nt * 8 * 32 * 8 : 0; }    // bytes per warp
constexpr int MAX_ENTRIES = 4096;
constexpr int ENTRY_ROWS = 256;               // packed query rows of a work list's item
constexpr float P_EXP = 15.f;                 // weights are w * 2^15
constexpr float P_UNIT = 1.f / 32768.f;
constexpr float VS_SPREAD = 100.f;            // log2 of the largest ratio of V scales that l holds

// A run that starts in a share and goes on in the next ones, for the kernel that joins its parts.
struct Cut {
  int parts;          // 0: the share has none
  int count, row, kvh;
  int64_t q0;
};

struct Work {
  Cut* cut;           // [workers]
  float* part_o;      // [2 workers][columns of a chunk][D]
  float4* part_ml;    // [2 workers][columns of a chunk]: m, l, log2 of the vs that l is relative to
  int workers;        // warps of the grid
  int entries;
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

// What an entry is, in shared memory: first unit on the line, keys that its rows see; for a work
// list also its runs, sequence, first query token and row, rows, and the keys before its first
// token (token j of the sequence's new ones sees keys [0, lo + j]).
template <bool LIST>
struct Entries {
  static constexpr int FIELDS = LIST ? 8 : 2;
  int n;
  int *cum, *lim, *runs, *seq, *q0, *row0, *rows, *lo;
  __device__ Entries(int* base, int n_) : n(n_) {
    cum = base;                                  // n + 1
    lim = cum + n + 1;
    if (LIST) {
      runs = lim + n;
      seq = runs + n;
      q0 = seq + n;
      row0 = q0 + n;
      rows = row0 + n;
      lo = rows + n;
    }
  }
  static size_t bytes(int n) { return (static_cast<size_t>(FIELDS) * n + 1) * sizeof(int); }
};

// Fills the entries; every thread of the CTA takes part.  HT: columns per chunk.  Returns the number
// of runs.
template <bool LIST, int HT>
__device__ int scan_entries(const Args& a, const Entries<LIST>& en, int* s_tot) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t cap = static_cast<int64_t>(a.bt_width) << a.log2_bs;
  int base = 0, total_runs = 0;
  for (int e0 = 0; e0 < en.n; e0 += THREADS) {
    const int e = e0 + tid;
    int lim = 0, runs = a.hkv * ((a.group + HT - 1) / HT);
    if (e < en.n) {
      int seq = e;
      if (LIST) {
        seq = a.tile_seq[e];
        const int row0 = a.tile_row0[e];
        if (seq >= a.num_seqs || row0 < 0) {
          record_error(a.err, kErrBounds);
          seq = -1;
        }
        int q0 = 0, rows = 0, lo = 0;
        if (seq >= 0) {
          q0 = a.cu_q[seq];
          int n = a.cu_q[seq + 1] - q0;
          if (q0 < 0 || n < 0 || n > a.tokens - q0) {
            record_error(a.err, kErrBounds);
            n = 0;
          }
          rows = max(0, min(n * a.group - row0, ENTRY_ROWS));
          lim = max(0, a.seq_lens[seq]);
          if (lim > cap) {
            record_error(a.err, kErrBounds);
            lim = static_cast<int>(cap);
          }
          lo = a.causal ? lim - n : 0x3fffffff;
          if (a.causal) lim = max(0, min(lim, lo + (row0 + rows - 1) / a.group + 1));
          if (rows == 0) lim = 0;
        }
        runs = a.hkv * ((rows + HT - 1) / HT);
        en.runs[e] = runs;
        en.seq[e] = seq;
        en.q0[e] = q0;
        en.row0[e] = row0;
        en.rows[e] = rows;
        en.lo[e] = lo;
      } else {
        lim = max(0, a.seq_lens[seq]);
        if (lim > cap) {
          record_error(a.err, kErrBounds);
          lim = static_cast<int>(cap);
        }
      }
      en.lim[e] = lim;
    }
    int v = (lim + KT - 1) / KT * runs;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += up;
    }
    const int r = __reduce_add_sync(0xffffffffu, lim > 0 ? runs : 0);
    if (lane == 31) {
      s_tot[warp] = v;
      s_tot[WARPS + warp] = r;
    }
    __syncthreads();
    int all = 0;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) v += s_tot[w];
      all += s_tot[w];
      total_runs += s_tot[WARPS + w];
    }
    if (e < en.n) en.cum[e + 1] = base + v;
    if (e == 0) en.cum[0] = 0;
    base += all;
    __syncthreads();
  }
  return total_runs;
}

// Shares: worker w of n takes units [w U / n, (w + 1) U / n).  While there are fewer tiles than the
// warps could take, a longer share costs its warp about a microsecond a tile and a shorter one gives
// the join more parts: sqrt(tiles of a run) / 4 tiles a share balances them.  us with 1 / 2 / 4 / 8 (8
// KV heads): 1 x 300 keys 7.7 / 8.4 / 11.6 / 16.5, 1 x 2047 11.7 / 10.4 / 11.9 / 16.2, 1 x 8000 27.4 /
// 19.4 / 16.8 / 18.9, 1 x 30000 35 / 35 / 35 / 29.
__device__ __forceinline__ int active_workers(int units, int runs, int workers) {
  const int tiles = max(1, __float2int_rn(0.25f * sqrtf(__fdividef(units, max(1, runs)))));
  return max(1, min(workers, units / tiles));
}
__device__ __forceinline__ int share_begin(int w, int units, int n) {
  return static_cast<int>(static_cast<int64_t>(w) * units / n);
}
__device__ __forceinline__ int share_of(int unit, int units, int n) {
  return static_cast<int>(((static_cast<int64_t>(unit) + 1) * n - 1) / units);
}

// A position on the line of tiles.
template <bool LIST>
struct Cursor {
  int e, r, t, nt;   // entry, run, tile, tiles of a run
  __device__ void seek(const Entries<LIST>& en, int unit) {
    int lo = 0, hi = en.n;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (en.cum[mid] <= unit) lo = mid;
      else hi = mid;
    }
    e = lo;
    nt = (en.lim[e] + KT - 1) / KT;
    const int x = unit - en.cum[e];
    r = x / nt;
    t = x - r * nt;
  }
  // to the next tile; only called when one exists
  __device__ void next(const Entries<LIST>& en, int runs) {
    if (++t < nt) return;
    t = 0;
    if (++r < (LIST ? en.runs[e] : runs)) return;
    r = 0;
    do ++e;
    while (en.cum[e + 1] == en.cum[e]);
    nt = (en.lim[e] + KT - 1) / KT;
  }
};

// The query rows of a run: column i is packed row `row + i` of the sequence's new tokens.
struct Columns {
  int kvh, seq, row, count, lo;
  int64_t q0;                  // first query token of the sequence
};
template <bool LIST, int HT>
__device__ __forceinline__ Columns columns_of(const Args& a, const Entries<LIST>& en,
                                              const Cursor<LIST>& c) {
  const int runs = LIST ? en.runs[c.e] : a.hkv * ((a.group + HT - 1) / HT);
  const int chunks = runs / a.hkv;
  Columns k;
  k.kvh = c.r / chunks;
  const int chunk = c.r - k.kvh * chunks;
  const int rows = LIST ? en.rows[c.e] : a.group;
  k.seq = LIST ? en.seq[c.e] : c.e;
  k.row = (LIST ? en.row0[c.e] : 0) + chunk * HT;
  k.count = min(HT, rows - chunk * HT);
  k.lo = LIST ? en.lo[c.e] : 0x3fffffff;
  k.q0 = LIST ? en.q0[c.e] : c.e;
  return k;
}

template <bool LIST, int NT>   // NT: column tiles of 8 per chunk
__global__ void __launch_bounds__(THREADS, ctas_of(NT))
    rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const Args a, const Work wk) {
  constexpr int HT = 8 * NT, STAGES = stages_of(NT), WARP_SMEM = STAGES * STAGE;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* ring = smem + warp * WARP_SMEM;
  constexpr bool Q_SMEM = q_smem_of(NT) > 0;
  constexpr int META = WARPS * (WARP_SMEM + q_smem_of(NT));
  uint2* s_q = reinterpret_cast<uint2*>(smem + WARPS * WARP_SMEM + warp * q_smem_of(NT)) + lane;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + META) + warp * STAGES;
  // scales of a stage's slices: [stage][slice][ks, vs]
  float* s_scale = reinterpret_cast<float*>(smem + META + WARPS * STAGES * 8) +
                   warp * STAGES * 4;
  int* s_tot = reinterpret_cast<int*>(smem + META + WARPS * STAGES * 24);
  const Entries<LIST> en(s_tot + 2 * WARPS, wk.entries);
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) mbar_init(&full[s], 3);   // lane 0's expect + two scale loads
    fence_barrier_init();
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  __syncwarp();
  pdl_trigger();
  const int w = warp * gridDim.x + blockIdx.x;   // neighbours on the line sit on different SMs
  if (lane == 0) wk.cut[w].parts = 0;
  const int all_runs = scan_entries<LIST, HT>(a, en, s_tot);
  // rows that see no key give 0
  for (int e = blockIdx.x; e < en.n; e += gridDim.x) {
    if (en.lim[e] > 0) continue;                                    // CTA-uniform
    const int row0 = LIST ? en.row0[e] : 0, rows = LIST ? en.rows[e] : a.group;
    for (int i = threadIdx.x; i < rows * a.hkv * (D / 8); i += THREADS) {
      const int c = i % (D / 8), x = i / (D / 8), r = row0 + x % rows, kvh = x / rows;
      *reinterpret_cast<uint4*>(a.out + (LIST ? en.q0[e] + r / a.group : e) * a.out_ld +
                                static_cast<int64_t>(kvh * a.group + r % a.group) * D + c * 8) =
          make_uint4(0, 0, 0, 0);
    }
  }
  const int units = en.cum[en.n];
  if (units == 0) return;
  const int runs = a.hkv * ((a.group + HT - 1) / HT);   // of a decode entry
  const int n_act = active_workers(units, all_runs, wk.workers);
  if (w >= n_act) return;
  const int u_begin = share_begin(w, units, n_act), u_end = share_begin(w + 1, units, n_act);
  if (u_begin >= u_end) return;

  const int g = lane >> 2, t4 = lane & 3;
  const uint64_t pol = policy_evict_first();
  // ---- producer state: lanes 0 and 1 own the tile's slices; the block id of the next tile to
  // issue is fetched one tile early ----
  Cursor<LIST> pc;
  pc.seek(en, u_begin);
  auto place = [&](int& seq, int& kvh) {
    seq = LIST ? en.seq[pc.e] : pc.e;
    kvh = pc.r / ((LIST ? en.runs[pc.e] : runs) / a.hkv);
  };
  int p_seq, p_kvh;
  place(p_seq, p_kvh);
  int pu = u_begin, p_id = 0;
  auto fetch_id = [&]() {
    const int key = pc.t * KT + lane * SL;
    if (lane < 2 && pu < u_end && key < en.lim[pc.e])
      p_id = a.tables[p_seq * a.bt_stride + (key >> a.log2_bs)];
  };
  auto issue = [&](int stage) {
    if (pu >= u_end) return;                                       // warp-uniform
    const int key0 = pc.t * KT, len = en.lim[pc.e];
    if (lane == 0)
      mbar_arrive_expect_tx(&full[stage], (len - key0 > SL ? 2 : 1) * 2 * SLICE);
    __syncwarp();
    if (lane < 2) {
      const int key = key0 + lane * SL;
      if (key < len) {
        const int blk = checked_block(a, p_id);
        const int bh = blk * a.hkv + p_kvh;
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
      pc.next(en, runs);
      if (pc.t == 0) place(p_seq, p_kvh);
      fetch_id();
    }
  };
  fetch_id();
#pragma unroll 1
  for (int s = 0; s < STAGES; ++s) issue(s);

  Cursor<LIST> cc;
  cc.seek(en, u_begin);
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
    // ---- tiles [t0, t1) of one run ----
    const int t0 = cc.t, t1 = min(cc.nt, t0 + u_end - u), len = en.lim[cc.e];
    const Columns co = columns_of<LIST, HT>(a, en, cc);
    uint32_t qf[Q_SMEM ? 1 : NT][8][2];
    float hs[NT][2];
    // where column i's row lies in q and out, and the keys that it sees
    auto token_of = [&](int i) { return LIST ? (co.row + i) / a.group : 0; };
    auto head_of = [&](int i) {
      return co.kvh * a.group + (LIST ? (co.row + i) % a.group : co.row + i);
    };
    int see[NT][2], see_min = len;
    if (LIST) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) see[n][j] = co.lo + token_of(n * 8 + 2 * t4 + j) + 1;
      see_min = min(len, co.lo + token_of(0) + 1);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint2 raw[8];
      const int col = n * 8 + g;
      const bool have = col < co.count;
      const bf16* qp = a.q + (co.q0 + token_of(col)) * a.q_ld +
                       static_cast<int64_t>(head_of(col)) * D + t4 * 4;
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
        const uint2 f = make_uint2(pack_f16x2(x.x * up, x.y * up), pack_f16x2(y.x * up, y.y * up));
        if (Q_SMEM) {
          s_q[(n * 8 + c) * 32] = f;
        } else {
          qf[Q_SMEM ? 0 : n][c][0] = f.x;
          qf[Q_SMEM ? 0 : n][c][1] = f.y;
        }
      }
      const float down = pow2i(-sh) * a.scale_log2;
      hs[n][0] = __shfl_sync(0xffffffffu, down, t4 * 8);
      hs[n][1] = __shfl_sync(0xffffffffu, down, t4 * 8 + 4);
    }
    float m[NT][2], l[NT][2], o[NT][8][4], lv_ref = 0.f;   // lv_ref: log2 of the first tile's vs
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int d = 0; d < 8; ++d) o[n][d][0] = o[n][d][1] = o[n][d][2] = o[n][d][3] = 0.f;
    }
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
      ok = __all_sync(0xffffffffu, mbar_wait(&full[stage], phase, nullptr));
      if (!ok) break;
      const int left = len - t * KT;                     // keys of this tile that exist
      const int nsl = left > SL ? 2 : 1;
      const float2 sc0 = *reinterpret_cast<const float2*>(s_scale + stage * 4);
      const float2 sc1 = nsl > 1 ? *reinterpret_cast<const float2*>(s_scale + stage * 4 + 2) : sc0;
      if (t == t0) lv_ref = sc0.y > 0.f ? lg2(sc0.y) : sc1.y > 0.f ? lg2(sc1.y) : 0.f;
      const float lv0 = sc0.y == 0.f ? lv_ref : lg2(sc0.y), lv1 = sc1.y == 0.f ? lv_ref : lg2(sc1.y);
      const float rv0 = ex2(fminf(lv_ref - lv0, VS_SPREAD) - P_EXP);
      const float rv1 = ex2(fminf(lv_ref - lv1, VS_SPREAD) - P_EXP);
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
            uint2 f, h;
            if (Q_SMEM) {
              f = s_q[(n * 8 + c) * 32];
              h = s_q[(n * 8 + c + 1) * 32];
            } else {
              f = make_uint2(qf[Q_SMEM ? 0 : n][c][0], qf[Q_SMEM ? 0 : n][c][1]);
              h = make_uint2(qf[Q_SMEM ? 0 : n][c + 1][0], qf[Q_SMEM ? 0 : n][c + 1][1]);
            }
            mma_f16(s[i][n], x[0], x[1], x[2], x[3], f.x, f.y);
            mma_f16(s[i][n], y[0], y[1], y[2], y[3], h.x, h.y);
          }
        }
        const float ks = i ? sc1.x : sc0.x, lv = i ? lv1 : lv0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float f0 = ks * hs[n][0], f1 = ks * hs[n][1];
          s[i][n][0] = fmaf(s[i][n][0], f0, lv);
          s[i][n][1] = fmaf(s[i][n][1], f1, lv);
          s[i][n][2] = fmaf(s[i][n][2], f0, lv);
          s[i][n][3] = fmaf(s[i][n][3], f1, lv);
        }
      }
      if (see_min - t * KT < KT) {
        // keys that a row does not see, or past the end: whatever their memory holds, their score
        // is -inf
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int key = i * SL + (x < 2 ? g : key_of_row(8 + g));
              const int lim = LIST ? min(len, see[n][x & 1]) - t * KT : left;
              if (key >= lim) s[i][n][x] = -INFINITY;
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
          const float top = safe - P_EXP;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            s[i][n][j] = ex2(s[i][n][j] - top);
            s[i][n][j + 2] = ex2(s[i][n][j + 2] - top);
          }
          l[n][j] = fmaf(s[0][n][j] + s[0][n][j + 2], rv0,
                         fmaf(s[1][n][j] + s[1][n][j + 2], rv1, l[n][j] * corr[n][j]));
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float c0 = corr[n][0], c1 = corr[n][1];
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
          uint32_t p[NT][2];
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            p[n][0] = transpose8(pack_f16x2(s[i][n][0], s[i][n][1]));
            p[n][1] = transpose8(pack_f16x2(s[i][n][2], s[i][n][3]));
          }
          const uint32_t base = v_addr + stage * STAGE + i * SLICE;
          auto add_v = [&](auto masked, uint32_t keep) {
#pragma unroll
            for (int c2 = 0; c2 < 8; c2 += 2) {
              uint32_t r[4], x[4];
              ldsm_t8(r, base + (((c2 + kchunk) ^ (vrow & 7)) << 4));
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t lo = masked ? r[2 * e] & keep : r[2 * e];
                const uint32_t hi = masked ? r[2 * e + 1] & keep : r[2 * e + 1];
                e4m3x4_to_f16(lo, x[0], x[2]);
                e4m3x4_to_f16(hi, x[1], x[3]);
#pragma unroll
                for (int n = 0; n < NT; ++n)
                  mma_f16(o[n][c2 + e], x[0], x[1], x[2], x[3], p[n][0], p[n][1]);
              }
            }
          };
          if (left - i * SL >= SL) {
            add_v(std::false_type{}, 0u);
          } else {
            // codes of keys past the end become zeros (NaN times weight 0 would be NaN)
            uint32_t keep = 0;
#pragma unroll
            for (int y = 0; y < 4; ++y)
              if (key_of_row(2 * t4 + (y & 1) + (y & 2) * 4) < left - i * SL) keep |= 0xffu << (8 * y);
            add_v(std::true_type{}, keep);
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
    if (t0 == 0 && !whole && lane == 0)
      wk.cut[w] = Cut{share_of(u + cc.nt - 1, units, n_act) - w + 1, co.count, co.row, co.kvh, co.q0};
    const float v_ref = ex2(lv_ref);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const float l0 = sum_over_keys(l[n][0]), l1 = sum_over_keys(l[n][1]);
      const int h0 = n * 8 + 2 * t4;
      if (whole) {
        const float i0 = l0 != 0.f ? P_UNIT / l0 : 0.f, i1 = l1 != 0.f ? P_UNIT / l1 : 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (h0 + j >= co.count) continue;
          bf16* dst = a.out + (co.q0 + token_of(h0 + j)) * a.out_ld +
                      static_cast<int64_t>(head_of(h0 + j)) * D + g;
          const float inv = j ? i1 : i0;
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            dst[d * 16] = __float2bfloat16(o[n][d][j] * inv * v_ref);
            dst[d * 16 + 8] = __float2bfloat16(o[n][d][j + 2] * inv * v_ref);
          }
        }
      } else {
        float* dst = wk.part_o + (static_cast<int64_t>(slot) * HT + h0) * D + g;
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          dst[d * 16] = o[n][d][0];
          dst[d * 16 + 8] = o[n][d][2];
          dst[D + d * 16] = o[n][d][1];
          dst[D + d * 16 + 8] = o[n][d][3];
        }
        if (g == 0) {
          wk.part_ml[slot * HT + h0] = make_float4(m[n][0], l0, lv_ref, 0.f);
          wk.part_ml[slot * HT + h0 + 1] = make_float4(m[n][1], l1, lv_ref, 0.f);
        }
      }
    }
    u += t1 - t0;
    if (u < u_end) {
      cc.t = cc.nt - 1;
      cc.next(en, runs);
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

// Joins the parts of the runs that share boundaries cut, in the order of the keys.  One warp per
// (share, column): the share that a cut run starts in describes it.  The parts' maxima and sums are
// read by the lanes together, their O rows (4 dims per lane) eight at a time.  The sums are brought to
// the first part's vs; the two factors are applied one after the other, since each alone fits 2^+-100.
template <bool LIST, int NT>
__global__ void __launch_bounds__(THREADS) join_kernel(const Args a, const Work wk) {
  constexpr int HT = 8 * NT;
  const int lane = threadIdx.x & 31;
  const int i = blockIdx.x * WARPS + (threadIdx.x >> 5);
  const int w = i / HT, col = i % HT;
  pdl_trigger();
  pdl_wait();
  if (w >= wk.workers) return;
  const Cut cut = wk.cut[w];
  if (col >= cut.count || cut.parts == 0) return;
  auto row_of = [&](int k) {
    return static_cast<int64_t>(k == 0 ? 2 * w + 1 : 2 * (w + k)) * HT + col;
  };
  float m = -INFINITY;
  for (int k = lane; k < cut.parts; k += 32) m = fmaxf(m, wk.part_ml[row_of(k)].x);
  m = warp_max(m);
  const float safe = m == -INFINITY ? 0.f : m;
  const float lv_ref = wk.part_ml[row_of(0)].z;
  float o[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
  for (int k0 = 0; k0 < cut.parts; k0 += 32) {
    const int n = min(32, cut.parts - k0);
    float f = 0.f;
    if (lane < n) {
      const float4 ml = wk.part_ml[row_of(k0 + lane)];
      f = ex2(ml.x - safe);
      l += ml.y * f * ex2(fminf(lv_ref - ml.z, VS_SPREAD));
    }
    for (int k = 0; k < n; k += 8) {
      float4 v[8];
#pragma unroll
      for (int x = 0; x < 8; ++x)
        v[x] = k + x < n
                   ? *reinterpret_cast<const float4*>(wk.part_o + row_of(k0 + k + x) * D + lane * 4)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const float c = __shfl_sync(0xffffffffu, f, (k + x) & 31);
        if (k + x < n) {
          o[0] += v[x].x * c;
          o[1] += v[x].y * c;
          o[2] += v[x].z * c;
          o[3] += v[x].w * c;
        }
      }
    }
  }
  l = warp_sum(l);
  const float inv = l != 0.f ? P_UNIT / l : 0.f, v_ref = ex2(lv_ref);
  const int tok = LIST ? (cut.row + col) / a.group : 0;
  const int head = cut.kvh * a.group + (LIST ? (cut.row + col) % a.group : cut.row + col);
  *reinterpret_cast<uint2*>(a.out + (cut.q0 + tok) * a.out_ld + static_cast<int64_t>(head) * D +
                            lane * 4) =
      make_uint2(pack_bf16x2(o[0] * inv * v_ref, o[1] * inv * v_ref),
                 pack_bf16x2(o[2] * inv * v_ref, o[3] * inv * v_ref));
}

// Upper bound of the line's length.
static int64_t line_bound(const Args& a, bool list, int ht) {
  const int64_t rows = list ? ENTRY_ROWS : a.group;
  return (list ? a.num_tiles : a.num_seqs) * static_cast<int64_t>(a.hkv) * ((rows + ht - 1) / ht) *
         (((static_cast<int64_t>(a.bt_width) << a.log2_bs) + KT - 1) / KT);
}

template <bool LIST, int NT>
void launch(const Args& a, const CUtensorMap& tk, const CUtensorMap& tv, const at::Tensor& like,
            cudaStream_t st) {
  constexpr int HT = 8 * NT, STAGES = stages_of(NT), WARP_SMEM = STAGES * STAGE;
  Work wk;
  wk.entries = LIST ? a.num_tiles : a.num_seqs;
  const size_t lens = 2 * WARPS * sizeof(int) + Entries<LIST>::bytes(wk.entries);
  const size_t smem = 1024 + WARPS * (WARP_SMEM + q_smem_of(NT)) + WARPS * STAGES * 24 + lens;
  static std::atomic<bool> allowed[64] = {};
  allow_smem(rows_kernel<LIST, NT>, 227 * 1024, allowed);
  // fewer CTAs an SM when the entries' tables of a very large batch need the room; no more warps
  // than the tiles there can be make shares
  const int per_sm = std::max<int>(1, std::min<size_t>(ctas_of(NT), 228 * 1024 / (smem + 1024)));
  const int64_t tiles = line_bound(a, LIST, HT);
  const int grid = static_cast<int>(
      std::max<int64_t>(1, std::min<int64_t>(148 * per_sm, (tiles + WARPS - 1) / WARPS)));
  wk.workers = grid * WARPS;
  static_assert(sizeof(Cut) % 8 == 0, "the cuts follow the partials");
  const int64_t part_rows = static_cast<int64_t>(wk.workers) * 2 * HT;
  at::Tensor ws = at::empty({wk.workers * static_cast<int64_t>(sizeof(Cut) / 4) + part_rows * (D + 4)},
                            like.options().dtype(at::kFloat));
  wk.part_o = ws.data_ptr<float>();
  wk.part_ml = reinterpret_cast<float4*>(wk.part_o + part_rows * D);
  wk.cut = reinterpret_cast<Cut*>(wk.part_ml + part_rows);
  auto rk = rows_kernel<LIST, NT>;
  auto jk = join_kernel<LIST, NT>;
  // A plain launch, after the previous kernel has left every SM: started early (programmatic
  // launch), CTAs fill the SMs around the previous kernel's last ones unevenly, and with equal shares
  // the fullest SM decides (256 x 2304: 163 us against 125).
  rk<<<grid, THREADS, smem, st>>>(tk, tv, a, wk);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  C10_CUDA_CHECK(launch_k(jk, dim3(wk.workers * HT / WARPS), dim3(THREADS), 0, st, nullptr, 0, a, wk));
}

}  // namespace fp8d

bool fp8_rows_fits(const fp8a::Args& a, bool list) {
  return (list ? a.num_tiles : a.num_seqs) <= fp8d::MAX_ENTRIES &&
         fp8d::line_bound(a, list, 8) < (int64_t(1) << 31);
}

void fp8_rows(const fp8a::Args& a, bool list, int64_t rows, const CUtensorMap& tk,
              const CUtensorMap& tv, const at::Tensor& like, cudaStream_t st) {
  using namespace fp8d;
  // As many column tiles as hold a decode group (16 columns at a time beyond that), or a list's items,
  // so that one pass over the keys does.  Lists of 64 items over 4000 keys, us with 1 / 2 /
  // 3 column tiles: 8 rows 95 / 103 / 132, 12 rows 179 / 104 / 133, 20 rows 268 / 189 / 136, 32 rows
  // 350 / 193 / 246 (two passes of 16 beat 24 + 8).
  if (list && (rows > 24 || (rows > 8 && rows <= 16))) launch<true, 2>(a, tk, tv, like, st);
  else if (list && rows > 16) launch<true, 3>(a, tk, tv, like, st);
  else if (list) launch<true, 1>(a, tk, tv, like, st);
  else if (a.group <= 8) launch<false, 1>(a, tk, tv, like, st);
  else launch<false, 2>(a, tk, tv, like, st);
}

}  // namespace lb
