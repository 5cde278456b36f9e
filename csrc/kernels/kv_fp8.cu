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
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>

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
  float norm_dim, eps;
  int T, hq, hkv, bs, num_blocks;
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
__device__ __forceinline__ float exp2i(int k) { return __uint_as_float((k + 127) << 23); }

// Row t's head at src, 4 elements per lane: optional RMSNorm, then the rotation.  Products and
// sums are rounded one by one, as the formula's separate operations are.
__device__ __forceinline__ void load_rotated(const Args& a, const bf16* src, int t, int lane,
                                             const bf16* nw, bool rotate, float (&o)[4]) {
  const uint2 raw = *reinterpret_cast<const uint2*>(src + lane * 4);
  const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
  const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
  float v[4] = {x.x, x.y, y.x, y.y};
  if (nw != nullptr) {
    const float ss = warp_sum(v[0] * v[0] + v[1] * v[1] + v[2] * v[2] + v[3] * v[3]);
    const float inv = rsqrtf(ss / a.norm_dim + a.eps);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = __fmul_rn(__fmul_rn(v[i], inv), __bfloat162float(nw[lane * 4 + i]));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = v[i];
  if (!rotate) return;
  int pos = a.positions[t];
  if (static_cast<unsigned>(pos) >= static_cast<unsigned>(a.max_pos)) {
    if (lane == 0) record_error(a.err, kErrBounds);
    pos = 0;
  }
  const int half = a.rot >> 1, e0 = lane * 4;
  const bool rot = e0 < a.rot, first = e0 < half;
  const int plane = !rot ? lane : (first ? lane + (half >> 2) : lane - (half >> 2));
  float p[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) p[i] = __shfl_sync(0xffffffffu, v[i], plane);
  if (rot) {
    const float* cs = a.cos_sin + static_cast<size_t>(pos) * a.rot + (first ? e0 : e0 - half);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float c = cs[i], s = cs[half + i];
      o[i] = first ? __fsub_rn(__fmul_rn(v[i], c), __fmul_rn(p[i], s))
                   : __fadd_rn(__fmul_rn(p[i], s), __fmul_rn(v[i], c));
    }
  }
}

__global__ void __launch_bounds__(THREADS) rope_kv_fp8_kernel(const Args a) {
  pdl_trigger();
  pdl_wait();
  const int heads = a.hq + 2 * a.hkv;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * (THREADS / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (w >= static_cast<int64_t>(a.T) * heads) return;      // warp-uniform
  const int t = static_cast<int>(w / heads), h = static_cast<int>(w % heads);
  if (h < a.hq) {
    float o[4];
    load_rotated(a, a.qkv + t * a.ld + h * D, t, lane, a.q_norm, true, o);
    const uint2 out = make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
    *reinterpret_cast<uint2*>(a.q_out + t * a.q_ld + h * D + lane * 4) = out;
    return;
  }
  // k or v head: the warp of the first row that goes to a block handles all of its rows
  const int slot = a.slots[t];
  if (slot < 0) return;
  const int blk = slot / a.bs;
  if (blk >= a.num_blocks) {
    if (lane == 0) record_error(a.err, kErrBounds);
    return;
  }
  for (int i = 0; i < a.bs - 1; i += 32) {
    const int r = t - 1 - i - lane;
    const int s = r >= 0 && i + lane < a.bs - 1 ? a.slots[r] : -1;
    if (__any_sync(0xffffffffu, s >= 0 && s / a.bs == blk)) return;
  }
  const bool is_v = h >= a.hq + a.hkv;
  const int kh = is_v ? h - a.hq - a.hkv : h - a.hq;
  const bf16* nw = is_v ? nullptr : a.k_norm;
  const int end = min(a.T, t + a.bs);
  float amax = 0.f;
  for (int r = t; r < end; ++r) {
    const int s = a.slots[r];
    if (s < 0 || s / a.bs != blk) continue;
    float o[4];
    load_rotated(a, a.qkv + r * a.ld + h * D, r, lane, nw, !is_v, o);
#pragma unroll
    for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fabsf(o[i]));
  }
  amax = warp_max(amax);
  float* sp = (is_v ? a.v_scale : a.k_scale) + static_cast<int64_t>(blk) * a.hkv + kh;
  uint8_t* base = (is_v ? a.v_cache : a.k_cache) +
                  (static_cast<int64_t>(blk) * a.hkv + kh) * a.bs * D;
  const int first = slot - blk * a.bs;
  float scale = exp2i(scale_exp(amax));
  if (first > 0) {
    const float old = *sp;
    if (old >= scale) {
      scale = old;
    } else {
      const float ratio = old / scale;
      for (int r = 0; r < first; ++r) {
        uint32_t* p = reinterpret_cast<uint32_t*>(base + r * D) + lane;
        float o[4];
        e4m3x4_to_f32(*p, o);
        *p = e4m3x4(o[0] * ratio, o[1] * ratio, o[2] * ratio, o[3] * ratio);
      }
    }
  }
  const float inv = 1.f / scale;
  for (int r = t; r < end; ++r) {
    const int s = a.slots[r];
    if (s < 0 || s / a.bs != blk) continue;
    float o[4];
    load_rotated(a, a.qkv + r * a.ld + h * D, r, lane, nw, !is_v, o);
    *(reinterpret_cast<uint32_t*>(base + (s - blk * a.bs) * D) + lane) =
        e4m3x4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  }
  __syncwarp();
  if (lane == 0) *sp = scale;
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

void rope_kv_fp8(const at::Tensor& qkv, const at::Tensor& positions, const at::Tensor& slots,
                 const at::Tensor& cos_sin, at::Tensor& k_cache, at::Tensor& v_cache,
                 at::Tensor& k_scale, at::Tensor& v_scale, at::Tensor& q_out, int64_t hq,
                 int64_t hkv, const c10::optional<at::Tensor>& q_norm,
                 const c10::optional<at::Tensor>& k_norm, int64_t norm_dim, double eps,
                 at::Tensor& err) {
  using namespace kq;
  check_fp8_cache("rope_kv_fp8", k_cache, v_cache, k_scale, v_scale);
  const int64_t T = qkv.size(0), R = cos_sin.size(1);
  TORCH_CHECK(hq >= 1 && hkv >= 1 && k_cache.size(1) == hkv, "rope_kv_fp8: head counts");
  TORCH_CHECK(qkv.is_cuda() && qkv.dim() == 2 && qkv.scalar_type() == at::kBFloat16 &&
                  qkv.size(1) >= (hq + 2 * hkv) * D && (T <= 1 || qkv.stride(0) % 8 == 0) &&
                  qkv.stride(1) == 1 && reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0,
              "rope_kv_fp8: qkv bf16 [T, (hq + 2 hkv) 128], 16-byte aligned rows");
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
  if (T == 0) return;
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
  a.norm_dim = norm_dim > 0 ? static_cast<float>(norm_dim) : static_cast<float>(R);
  a.eps = static_cast<float>(eps);
  a.T = T;
  a.hq = hq;
  a.hkv = hkv;
  a.bs = k_cache.size(2);
  a.num_blocks = k_cache.size(0);
  a.err = err.data_ptr<int>();
  const int64_t warps = T * (hq + 2 * hkv);
  C10_CUDA_CHECK(launch_k(rope_kv_fp8_kernel, dim3((warps + THREADS / 32 - 1) / (THREADS / 32)),
                          dim3(THREADS), 0, at::cuda::getCurrentCUDAStream(), nullptr, 0, a));
}

}  // namespace lb
