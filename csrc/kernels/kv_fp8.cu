// RoPE and the quantised append to the 8-bit paged KV cache (sm_100a).
//
// The cache holds e4m3 codes [blocks, KV heads, BS, 128] and one fp32 scale per (block, KV head)
// for K and for V; a stored value is code * scale.  Scales are powers of two: with
//   s = 2^ceil(log2(amax / 448)), clamped to [2^-40, 2^119],
// amax / s lies in (224, 448], and when a later token of the block needs a larger scale s' the
// older codes are multiplied by s / s', which only moves their exponents: nothing is rounded
// twice unless a value falls below e4m3's smallest step (2^-9 of the new scale).  A scale
// amax / 448 would round every older code again at each growth and buys at most one bit of the
// range below the normal numbers.  A block entered at offset 0 takes its scale from this call's
// tokens alone (what it held belongs to a former owner).
//
// k and v are rounded once, from fp32 after norm and rotation.
//
// HBM traffic is qkv in, q and codes out (167 MB for 7.1k rows of 32 + 8 + 8 heads: 25.9 us at the
// measured copy rate); instructions bind it first.  Measured: 7.1k rows with norms 45.5 us (3.7 TB/s,
// 57 %), 256 decode rows 4.1 us, one row 3.0 us.  Tried: a warp holding 16 rows of a block 92 us
// (spills), lanes exchanging rotation partners by shuffle 65 us, 8 q heads per warp 49 us.
#include <ATen/Functions.h>
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include "checks.h"
#include "common.cuh"

namespace lb {
namespace kq {

constexpr int D = 128;
constexpr int THREADS = 128;
constexpr int MIN_EXP = -40, MAX_EXP = 119;

struct Args {
  const bf16* qkv;
  int64_t ld;
  const int* positions;
  const int* slots;
  const float* cos_sin;
  int max_pos, rot;
  bf16* q_out;
  int64_t q_ld;
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* k_scale;
  float* v_scale;
  const bf16* q_norm;
  const bf16* k_norm;
  float inv_norm_dim, eps;
  int T, hq, hkv, num_blocks;
  int* err;
};

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
__device__ __forceinline__ void e4m3x4_to_f32(uint32_t v, float (&o)[4]) {
  uint32_t lo, hi;
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(v));
  const float2 x = __half22float2(*reinterpret_cast<__half2*>(&lo));
  const float2 y = __half22float2(*reinterpret_cast<__half2*>(&hi));
  o[0] = x.x; o[1] = x.y; o[2] = y.x; o[3] = y.y;
}

// Exponent of the smallest power-of-two scale that brings amax to 448 or below:
// 448 = 1.75 * 2^8, so one more when amax's mantissa exceeds 1.75.
__device__ __forceinline__ int scale_exp(float amax) {
  const uint32_t u = __float_as_uint(fminf(amax, 3.4e38f));
  const int k = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(MAX_EXP, max(MIN_EXP, k));
}
__device__ __forceinline__ float max_abs(float m, float a, float b) {
  return fmaxf(m, fmaxf(fabsf(a), fabsf(b)));
}
__device__ __forceinline__ float exp2i(int k) { return __uint_as_float((k + 127) << 23); }

// Half a warp holds one head row.  A lane owns both partners of its rotations: four dims from d0 and
// their partners from d1 = d0 + rot / 2, so nothing is exchanged between lanes; lanes past the
// rotary width hold two runs of four dims that pass through.  The instructions per element bound
// this kernel before HBM does, so the arithmetic runs on fp32 pairs (mul / add .f32x2).  Products
// and sums are rounded one by one, as the formula's separate operations are.
typedef uint64_t f2;
__device__ __forceinline__ f2 pack2(float lo, float hi) {
  f2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void unpack2(f2 v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f2 sub2(f2 a, f2 b) {
  f2 d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f2 widen(uint32_t bf16_pair) {
  return pack2(__uint_as_float(bf16_pair << 16), __uint_as_float(bf16_pair & 0xffff0000u));
}

struct Lane {
  int d0, d1;      // first dim of the two runs of four
  bool in;         // rotates
};
__device__ __forceinline__ Lane lane_of(const Args& a, int lane) {
  Lane r;
  const int hl = lane & 15, half = a.rot >> 1;
  r.in = hl * 4 < half;
  r.d0 = r.in ? hl * 4 : a.rot + 8 * (hl - (half >> 2));
  r.d1 = r.in ? half + hl * 4 : r.d0 + 4;
  return r;
}
__device__ __forceinline__ uint4 load_row(const bf16* p, const Lane& ro) {
  const uint2 x = *reinterpret_cast<const uint2*>(p + ro.d0);
  const uint2 y = *reinterpret_cast<const uint2*>(p + ro.d1);
  return make_uint4(x.x, x.y, y.x, y.y);
}
__device__ __forceinline__ void widen4(const uint4& raw, f2 (&v)[4]) {
  v[0] = widen(raw.x);
  v[1] = widen(raw.y);
  v[2] = widen(raw.z);
  v[3] = widen(raw.w);
}
struct Turn {      // cos and sin of a lane's four rotations
  f2 c[2] = {0, 0}, s[2] = {0, 0};
};
__device__ __forceinline__ void load_turn(const Args& a, const Lane& ro, int lane, int t, Turn& tu) {
  int pos = a.positions[t];
  if (static_cast<unsigned>(pos) >= static_cast<unsigned>(a.max_pos)) {
    if ((lane & 15) == 0) record_error(a.err, kErrBounds);
    pos = 0;
  }
  if (ro.in) {
    const float* p = a.cos_sin + static_cast<size_t>(pos) * a.rot + ro.d0;
    const float4 c = *reinterpret_cast<const float4*>(p);
    const float4 s = *reinterpret_cast<const float4*>(p + (a.rot >> 1));
    tu.c[0] = pack2(c.x, c.y);
    tu.c[1] = pack2(c.z, c.w);
    tu.s[0] = pack2(s.x, s.y);
    tu.s[1] = pack2(s.z, s.w);
  }
}
// In place; both halves of the warp take part.
__device__ __forceinline__ void norm_turn(const Args& a, const Lane& ro, const f2* w, const Turn& tu,
                                          f2 (&v)[4]) {
  if (w != nullptr) {
    f2 q = mul2(v[0], v[0]);
#pragma unroll
    for (int i = 1; i < 4; ++i) q = fma2(v[i], v[i], q);
    float lo, hi;
    unpack2(q, lo, hi);
    float ss = lo + hi;
#pragma unroll
    for (int m = 1; m < 16; m <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
    const float inv = rsqrtf(ss * a.inv_norm_dim + a.eps);
    const f2 inv2 = pack2(inv, inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = mul2(mul2(v[i], inv2), w[i]);
  }
  if (ro.in) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f2 x = v[i], y = v[i + 2];
      v[i] = sub2(mul2(x, tu.c[i]), mul2(y, tu.s[i]));
      v[i + 2] = add2(mul2(x, tu.s[i]), mul2(y, tu.c[i]));
    }
  }
}
__device__ __forceinline__ uint32_t bf16_pair(f2 v) {
  float lo, hi;
  unpack2(v, lo, hi);
  return pack_bf16x2(lo, hi);
}
__device__ __forceinline__ uint32_t codes4(f2 a, f2 b, f2 inv) {
  float x[4];
  unpack2(mul2(a, inv), x[0], x[1]);
  unpack2(mul2(b, inv), x[2], x[3]);
  return e4m3x4(x[0], x[1], x[2], x[3]);
}

// ---- q: a warp takes two rows and HPW heads; the rows' cos and sin stay in registers ----
constexpr int HPW = 4;
__device__ __forceinline__ void rotate_q(const Args& a, int64_t w, int lane) {
  const int groups = (a.hq + HPW - 1) / HPW;
  const int t = static_cast<int>(w / groups) * 2 + (lane >> 4);
  const int h0 = static_cast<int>(w % groups) * HPW;
  const Lane ro = lane_of(a, lane);
  const bool live = t < a.T;
  const int n = live ? min(HPW, a.hq - h0) : 0;
  const bf16* src = a.qkv + t * a.ld + h0 * D;
  uint4 raw[HPW];
#pragma unroll
  for (int i = 0; i < HPW; ++i)
    raw[i] = i < n ? load_row(src + i * D, ro) : make_uint4(0, 0, 0, 0);
  Turn tu;
  if (live) load_turn(a, ro, lane, t, tu);
  f2 nw[4];
  const bool norm = a.q_norm != nullptr;
  if (norm) widen4(load_row(a.q_norm, ro), nw);
  bf16* dst = a.q_out + t * a.q_ld + h0 * D;
#pragma unroll
  for (int i = 0; i < HPW; ++i) {
    f2 v[4];
    widen4(raw[i], v);
    norm_turn(a, ro, norm ? nw : nullptr, tu, v);
    if (i < n) {
      *reinterpret_cast<uint2*>(dst + i * D + ro.d0) = make_uint2(bf16_pair(v[0]), bf16_pair(v[1]));
      *reinterpret_cast<uint2*>(dst + i * D + ro.d1) = make_uint2(bf16_pair(v[2]), bf16_pair(v[3]));
    }
  }
}

// ---- k, v: NW warps take the blocks that are entered in `win` consecutive rows, HPK heads ----
//
// The slots of the window and of BS rows on both sides sit in the lanes (row base + 32 k + lane in
// sl[k]); a ballot per block gives its rows.  A block belongs to the window that holds its first
// row.  Rows are rotated into registers four at a time per warp (two per step, half a warp each):
// while a block's rows fit the NW warps they are read once, otherwise twice (maximum, then codes).
constexpr int HPK = 2;
template <int BS, int NW>
__device__ __forceinline__ void append_kv(const Args& a, int64_t w, int win, int warp, int lane,
                                          float (*s_max)[HPK]) {
  constexpr int NR = (2 * BS + 16 + 31) / 32;
  const int groups = (a.hkv + HPK - 1) / HPK;
  const int w0 = static_cast<int>(w / (2 * groups)) * win, gi = static_cast<int>(w % (2 * groups));
  const bool is_v = gi >= groups;
  const int kh0 = (is_v ? gi - groups : gi) * HPK;
  const int base = w0 - BS;
  int sl[NR];
#pragma unroll
  for (int k = 0; k < NR; ++k) {
    const int r = base + 32 * k + lane;
    sl[k] = r >= 0 && r < a.T ? a.slots[r] : -1;
  }
  const Lane ro = lane_of(a, lane);
  const bool norm = !is_v && a.k_norm != nullptr;
  f2 nw[4];
  if (norm) widen4(load_row(a.k_norm, ro), nw);
  // rows of the window that have a slot
  const int i0 = BS, i1 = BS + min(win, a.T - w0);
  uint32_t todo[NR];
#pragma unroll
  for (int k = 0; k < NR; ++k)
    todo[k] = __ballot_sync(0xffffffffu, sl[k] >= 0 && 32 * k + lane >= i0 && 32 * k + lane < i1);
  const bf16* head =
      a.qkv + static_cast<int64_t>(a.hq + (is_v ? a.hkv : 0) + kh0) * D;
  float* scales = is_v ? a.v_scale : a.k_scale;
  uint8_t* cache = is_v ? a.v_cache : a.k_cache;
  while (true) {
    int first = -1, slot = 0;
#pragma unroll
    for (int k = NR - 1; k >= 0; --k)
      if (todo[k]) {
        first = 32 * k + __ffs(todo[k]) - 1;
        slot = __shfl_sync(0xffffffffu, sl[k], first & 31);
      }
    if (first < 0) break;
    const int blk = slot / BS;
    bool earlier = false;
    int last = first;
#pragma unroll
    for (int k = 0; k < NR; ++k) {
      const int i = 32 * k + lane;
      const bool same = sl[k] >= 0 && sl[k] / BS == blk;
      earlier |= __any_sync(0xffffffffu, same && i < first && i > first - BS) != 0;
      const uint32_t mem = __ballot_sync(0xffffffffu, same && i >= first && i < first + BS);
      todo[k] &= ~mem;
      if (mem) last = 32 * k + 31 - __clz(mem);
    }
    if (earlier) continue;                          // another window's block
    if (blk >= a.num_blocks) {
      if (lane == 0) record_error(a.err, kErrBounds);
      continue;
    }
    const int row_a = base + first, row_b = base + last;
    const int chunks = (row_b - row_a + 4 * NW) / (4 * NW);
    const int64_t bh = static_cast<int64_t>(blk) * a.hkv + kh0;
    float old[HPK];
#pragma unroll
    for (int h = 0; h < HPK; ++h) old[h] = kh0 + h < a.hkv ? scales[bh + h] : 0.f;
    f2 v[2][HPK][4];
    int off[2];                                     // the row's place in the block, -1: none
    auto load = [&](int c) {
      uint4 raw[2][HPK];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = row_a + (c * NW + warp) * 4 + 2 * i + (lane >> 4);
        const int x = row <= row_b ? a.slots[row] : -1;
        off[i] = x >= 0 && x / BS == blk ? x - blk * BS : -1;
#pragma unroll
        for (int h = 0; h < HPK; ++h)
          raw[i][h] = off[i] >= 0 && kh0 + h < a.hkv
                          ? load_row(head + row * a.ld + h * D, ro)
                          : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int h = 0; h < HPK; ++h) widen4(raw[i][h], v[i][h]);
        if (!is_v) {
          const int row = row_a + (c * NW + warp) * 4 + 2 * i + (lane >> 4);
          Turn tu;
          if (off[i] >= 0) load_turn(a, ro, lane, row, tu);
#pragma unroll
          for (int h = 0; h < HPK; ++h) norm_turn(a, ro, norm ? nw : nullptr, tu, v[i][h]);
        }
      }
    };
    float amax[HPK];
#pragma unroll
    for (int h = 0; h < HPK; ++h) amax[h] = 0.f;
    for (int c = 0; c < chunks; ++c) {
      load(c);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < HPK; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float lo, hi;
            unpack2(v[i][h][e], lo, hi);
            amax[h] = max_abs(amax[h], lo, hi);
          }
    }
#pragma unroll
    for (int h = 0; h < HPK; ++h) amax[h] = warp_max(amax[h]);
    if (NW > 1) {
      __syncthreads();                              // s_max of the previous block has been read
      if (lane == 0) {
#pragma unroll
        for (int h = 0; h < HPK; ++h) s_max[warp][h] = amax[h];
      }
      __syncthreads();                              // and every warp has read the old scales
#pragma unroll
      for (int h = 0; h < HPK; ++h)
#pragma unroll
        for (int k = 0; k < NW; ++k) amax[h] = fmaxf(amax[h], s_max[k][h]);
    }
    const int entry = slot - blk * BS;
    float inv[HPK];
#pragma unroll
    for (int h = 0; h < HPK; ++h) {
      if (kh0 + h >= a.hkv) continue;
      float scale = exp2i(scale_exp(amax[h]));
      if (entry > 0) {
        if (old[h] >= scale) {
          scale = old[h];
        } else {
          const float ratio = old[h] / scale;
          for (int r = warp * 2 + (lane >> 4); r < entry; r += 2 * NW) {
            uint8_t* p = cache + ((bh + h) * BS + r) * D;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t* x = reinterpret_cast<uint32_t*>(p + (e ? ro.d1 : ro.d0));
              float f[4];
              e4m3x4_to_f32(*x, f);
              *x = e4m3x4(f[0] * ratio, f[1] * ratio, f[2] * ratio, f[3] * ratio);
            }
          }
        }
      }
      inv[h] = 1.f / scale;
      __syncwarp();                                 // NW == 1: every lane has read the old scale
      if (warp == 0 && lane == 0) scales[bh + h] = scale;
    }
    for (int c = chunks - 1; c >= 0; --c) {
      if (c != chunks - 1) load(c);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int h = 0; h < HPK; ++h)
          if (off[i] >= 0 && kh0 + h < a.hkv) {
            const f2 s = pack2(inv[h], inv[h]);
            uint8_t* p = cache + ((bh + h) * BS + off[i]) * D;
            *reinterpret_cast<uint32_t*>(p + ro.d0) = codes4(v[i][h][0], v[i][h][1], s);
            *reinterpret_cast<uint32_t*>(p + ro.d1) = codes4(v[i][h][2], v[i][h][3], s);
          }
    }
  }
}

template <int BS, int NW>
__global__ void __launch_bounds__(THREADS, 5) rope_kv_fp8_kernel(const Args a, int win,
                                                              int kv_ctas) {
  __shared__ float s_max[THREADS / 32][HPK];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int WPC = THREADS / 32;
  if (static_cast<int>(blockIdx.x) < kv_ctas) {
    const int64_t items = static_cast<int64_t>((a.T + win - 1) / win) * 2 * ((a.hkv + HPK - 1) / HPK);
    const int64_t w = static_cast<int64_t>(blockIdx.x) * (WPC / NW) + warp / NW;
    if (w < items) append_kv<BS, NW>(a, w, win, warp % NW, lane, s_max);
  } else {
    const int64_t w = static_cast<int64_t>(blockIdx.x - kv_ctas) * WPC + warp;
    if (w < static_cast<int64_t>((a.T + 1) / 2) * ((a.hq + HPW - 1) / HPW)) rotate_q(a, w, lane);
  }
}

}  // namespace kq

// The fp8 cache's layout, shared by the append and the attention.
void check_fp8_cache(const char* op, const at::Tensor& k_cache, const at::Tensor& v_cache,
                     const at::Tensor& k_scale, const at::Tensor& v_scale) {
  TORCH_CHECK(k_cache.is_cuda() && k_cache.scalar_type() == at::kFloat8_e4m3fn &&
                  v_cache.scalar_type() == at::kFloat8_e4m3fn && k_cache.dim() == 4 &&
                  k_cache.is_contiguous() && v_cache.is_contiguous() &&
                  k_cache.sizes() == v_cache.sizes() && k_cache.size(3) == 128,
              op, ": caches are contiguous float8_e4m3fn [num_blocks, Hkv, block size, 128]");
  check_same_device(op, k_cache, {&v_cache, &k_scale, &v_scale});
  const int64_t bs = k_cache.size(2);
  TORCH_CHECK(bs == 16 || bs == 32 || bs == 64, op, ": block size 16, 32 or 64");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(k_cache.data_ptr()) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(v_cache.data_ptr()) % 16 == 0,
              op, ": caches start on 16-byte boundaries");
  for (const at::Tensor* s : {&k_scale, &v_scale})
    TORCH_CHECK(s->is_cuda() && s->scalar_type() == at::kFloat && s->is_contiguous() &&
                    s->dim() == 2 && s->size(0) == k_cache.size(0) && s->size(1) == k_cache.size(1),
                op, ": scales are contiguous float32 [num_blocks, Hkv]");
  // Slots and the TMA row coordinates ((block * Hkv + head) * BS + key) are int32.
  TORCH_CHECK(k_cache.size(0) * k_cache.size(1) * bs < (int64_t(1) << 31), op,
              ": KV pool rows exceed int32");
}

at::Tensor rope_kv_fp8(const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& slots,
                       const at::Tensor& cos_sin, at::Tensor& k_cache, at::Tensor& v_cache,
                       at::Tensor& k_scale, at::Tensor& v_scale,
                       const c10::optional<at::Tensor>& out, int64_t hq, int64_t hkv,
                       const c10::optional<at::Tensor>& q_norm,
                       const c10::optional<at::Tensor>& k_norm, int64_t norm_dim, double eps,
                       at::Tensor& err) {
  using namespace kq;
  check_fp8_cache("rope_kv_fp8", k_cache, v_cache, k_scale, v_scale);
  auto given = [](const c10::optional<at::Tensor>& t) {
    return t.has_value() && t->defined() ? &*t : nullptr;
  };
  check_same_device("rope_kv_fp8", k_cache, {&qkv, &positions, &slots, &cos_sin, &err, given(out),
                                             given(q_norm), given(k_norm)});
  const c10::cuda::CUDAGuard guard(k_cache.device());
  const int64_t T = qkv.size(0), R = cos_sin.size(1);
  TORCH_CHECK(hq >= 1 && hkv >= 1 && k_cache.size(1) == hkv, "rope_kv_fp8: head counts");
  TORCH_CHECK(qkv.is_cuda() && qkv.dim() == 2 && qkv.scalar_type() == at::kBFloat16 &&
                  qkv.size(1) >= (hq + 2 * hkv) * D && (T <= 1 || qkv.stride(0) % 8 == 0) &&
                  qkv.stride(1) == 1 && reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0,
              "rope_kv_fp8: qkv bf16 [T, (hq + 2 hkv) 128], 16-byte aligned rows");
  at::Tensor q_out =
      out.has_value() && out->defined() ? *out : at::empty({T, hq, D}, qkv.options());
  TORCH_CHECK(q_out.is_cuda() && q_out.scalar_type() == at::kBFloat16 && q_out.dim() == 3 &&
                  q_out.size(0) == T && q_out.size(1) == hq && q_out.size(2) == D &&
                  q_out.stride(2) == 1 && q_out.stride(1) == D &&
                  (T <= 1 || q_out.stride(0) % 8 == 0) &&
                  reinterpret_cast<uintptr_t>(q_out.data_ptr()) % 16 == 0,
              "rope_kv_fp8: q_out bf16 [T, hq, 128], contiguous heads, 16-byte aligned rows");
  TORCH_CHECK(positions.is_cuda() && positions.scalar_type() == at::kInt &&
                  positions.is_contiguous() && positions.numel() >= T && slots.is_cuda() &&
                  slots.scalar_type() == at::kInt && slots.is_contiguous() && slots.numel() >= T,
              "rope_kv_fp8: positions and slots are contiguous int32 [T]");
  TORCH_CHECK(cos_sin.is_cuda() && cos_sin.dim() == 2 && cos_sin.scalar_type() == at::kFloat &&
                  cos_sin.is_contiguous() && cos_sin.size(0) >= 1 && R >= 16 && R <= D &&
                  R % 16 == 0 && reinterpret_cast<uintptr_t>(cos_sin.data_ptr()) % 16 == 0,
              "rope_kv_fp8: cos_sin float32 [positions, rotary width], a multiple of 16 up to 128");
  Args a;
  for (int i = 0; i < 2; ++i) {
    const c10::optional<at::Tensor>& w = i == 0 ? q_norm : k_norm;
    const bool has = w.has_value() && w->defined();
    if (has)
      TORCH_CHECK(w->is_cuda() && w->scalar_type() == at::kBFloat16 && w->is_contiguous() &&
                      w->numel() == D && reinterpret_cast<uintptr_t>(w->data_ptr()) % 16 == 0,
                  "rope_kv_fp8: q/k norm weights are bf16 [128]");
    (i == 0 ? a.q_norm : a.k_norm) =
        has ? reinterpret_cast<const bf16*>(w->data_ptr()) : nullptr;
  }
  if (T == 0) return q_out;
  a.qkv = reinterpret_cast<const bf16*>(qkv.data_ptr());
  a.ld = qkv.stride(0);
  a.positions = positions.data_ptr<int>();
  a.slots = slots.data_ptr<int>();
  a.cos_sin = cos_sin.data_ptr<float>();
  a.max_pos = static_cast<int>(std::min<int64_t>(cos_sin.size(0), INT32_MAX));
  a.rot = R;
  a.q_out = reinterpret_cast<bf16*>(q_out.data_ptr());
  a.q_ld = q_out.stride(0);
  a.k_cache = reinterpret_cast<uint8_t*>(k_cache.data_ptr());
  a.v_cache = reinterpret_cast<uint8_t*>(v_cache.data_ptr());
  a.k_scale = k_scale.data_ptr<float>();
  a.v_scale = v_scale.data_ptr<float>();
  a.inv_norm_dim = 1.f / (norm_dim > 0 ? static_cast<float>(norm_dim) : static_cast<float>(R));
  a.eps = static_cast<float>(eps);
  a.T = T;
  a.hq = hq;
  a.hkv = hkv;
  a.num_blocks = k_cache.size(0);
  a.err = err.data_ptr<int>();
  // A warp per row (and head pair) while that leaves the GPU room: a decode batch, every row its own
  // block.  Beyond that the rows are mostly chunks of prompts: four warps share a window of 16 rows,
  // which holds about one block, and read it once.
  constexpr int WPC = THREADS / 32;
  const int64_t pairs = 2 * ((hkv + HPK - 1) / HPK);
  const bool few = T * pairs <= 148 * 32;
  const int win = few ? 1 : 16;
  const int64_t kv = few ? (T * pairs + WPC - 1) / WPC : (T + 15) / 16 * pairs;
  const int64_t qw = ((T + 1) / 2 * ((hq + HPW - 1) / HPW) + WPC - 1) / WPC;
  TORCH_CHECK(kv + qw < (int64_t(1) << 31), "rope_kv_fp8: too many rows");
  const int64_t bs = k_cache.size(2);
  auto kernel = bs == 16   ? (few ? rope_kv_fp8_kernel<16, 1> : rope_kv_fp8_kernel<16, 4>)
                : bs == 32 ? (few ? rope_kv_fp8_kernel<32, 1> : rope_kv_fp8_kernel<32, 4>)
                           : (few ? rope_kv_fp8_kernel<64, 1> : rope_kv_fp8_kernel<64, 4>);
  C10_CUDA_CHECK(launch_k(kernel, dim3(kv + qw), dim3(THREADS), 0,
                          at::cuda::getCurrentCUDAStream(), nullptr, 0, a, win,
                          static_cast<int>(kv)));
  return q_out;
}

}  // namespace lb
