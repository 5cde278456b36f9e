// What the decode and prefill kernels over the 8-bit KV cache share.
#pragma once

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAException.h>

#include <atomic>

#include "common.cuh"

namespace lb {

CUtensorMap make_tmap_bf16_2d(const void* ptr, uint64_t inner, uint64_t outer,
                              uint64_t row_stride_bytes, uint32_t box_inner, uint32_t box_outer,
                              CUtensorMapSwizzle swz);

namespace fp8a {

constexpr int D = 128;          // head width
constexpr int SL = 16;          // keys per cache slice: every block is a whole number of them
constexpr int SLICE = SL * D;   // bytes

struct Args {
  const bf16* q;
  int64_t q_ld;
  bf16* out;
  int64_t out_ld;
  const float* k_scale;
  const float* v_scale;
  const int* tables;
  int64_t bt_stride;
  int bt_width;
  const int* seq_lens;
  const int* cu_q;        // prefill: token offsets and the work list
  const int* tile_seq;
  const int* tile_row0;
  int num_tiles;
  int hq, hkv, group, log2_bs, num_blocks, num_seqs;
  int tokens;             // rows of q and out
  int causal;
  float scale_log2;
  int* err;
};

// e4m3 pairs -> f16 pairs (exact: e4m3's 2^-9 .. 448 are f16 numbers).
__device__ __forceinline__ void e4m3x4_to_f16(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(v));
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// q enters the tensor cores as f16 (K's codes are exact there).  Each row is first scaled by a
// power of two that brings its largest element to [2^14, 2^15): bf16's 8 bits then fit f16's 11
// for every element down to 2^-32 of the largest.  Returns the exponent of that power.
__device__ __forceinline__ int q_shift(float amax) {
  const int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
  return amax > 0.f ? min(126, max(-112, 14 - e)) : 0;
}
__device__ __forceinline__ float pow2i(int k) { return __uint_as_float((k + 127) << 23); }

// Lets the kernel have `bytes` of dynamic shared memory on the current device, once per device.  `done` is
// set only after the attribute holds: no other host thread launches before, and a failure is tried again.
template <typename K>
inline void allow_smem(K* kernel, int bytes, std::atomic<bool> (&done)[64]) {
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 64 && done[dev].load(std::memory_order_acquire)) return;
  C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) done[dev].store(true, std::memory_order_release);
}

// Physical block of slice `s` (16 keys) of a sequence; an id outside the pool is reported and
// replaced by block 0, so every TMA coordinate stays inside the tensor map.
__device__ __forceinline__ int checked_block(const Args& a, int id) {
  if (static_cast<unsigned>(id) >= static_cast<unsigned>(a.num_blocks)) {
    record_error(a.err, kErrBounds);
    return 0;
  }
  return id;
}

}  // namespace fp8a

// Launch on the current stream; the tensor maps view the caches as rows of 128 bytes.
// fp8_rows (attn_fp8_rows.cu): few query rows per sequence, one token each (list = false) or the
// work list's.  fp8_prefill (attn_fp8_prefill.cu): the work list's 256-row items on tcgen05.
bool fp8_rows_fits(const fp8a::Args& a, bool list);
// rows: query rows of a work list's longest item (or their mean, where only that is known).
void fp8_rows(const fp8a::Args& a, bool list, int64_t rows, const CUtensorMap& tk,
              const CUtensorMap& tv, const at::Tensor& like, cudaStream_t st);
void fp8_prefill(const fp8a::Args& a, const CUtensorMap& tk, const CUtensorMap& tv,
                 cudaStream_t st);

}  // namespace lb
