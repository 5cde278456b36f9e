// Paged attention over the 8-bit KV cache (sm_100a).
//
//   s_j = scale * ks_{b(j)} * (q . k8_j),  p_j = exp(s_j - max s),
//   o   = sum_j p_j vs_{b(j)} v8_j / sum_j p_j
//
// One warp per (query token, head): lane l holds dims 4 l .. 4 l + 3, keys one after another
// with a running maximum and sum.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>

#include "attn_fp8.cuh"

namespace lb {

void check_fp8_cache(const char* op, const at::Tensor& k_cache, const at::Tensor& v_cache,
                     const at::Tensor& k_scale, const at::Tensor& v_scale);

namespace fp8a {

__device__ __forceinline__ void unpack4(uint32_t v, float (&o)[4]) {
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

__device__ void attend(const Args& a, const uint8_t* k_cache, const uint8_t* v_cache, int seq, int64_t tok, int head, int klim, int lane) {
  const int kvh = head / a.group;
  const uint2 raw = *reinterpret_cast<const uint2*>(a.q + tok * a.q_ld + head * D + lane * 4);
  const float2 qx = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
  const float2 qy = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  const int bs = 1 << a.log2_bs;
  klim = min(klim, a.bt_width * bs);
  for (int b = 0; b * bs < klim; ++b) {
    int blk = a.tables[seq * a.bt_stride + b];
    if (static_cast<unsigned>(blk) >= static_cast<unsigned>(a.num_blocks)) {
      if (lane == 0) record_error(a.err, kErrBounds);
      blk = 0;
    }
    const int64_t bh = static_cast<int64_t>(blk) * a.hkv + kvh;
    const float ks = a.k_scale[bh] * a.scale_log2, vs = a.v_scale[bh];
    const int n = min(bs, klim - b * bs);
    for (int j = 0; j < n; ++j) {
      float k[4], v[4];
      unpack4(*reinterpret_cast<const uint32_t*>(k_cache + ((bh << a.log2_bs) + j) * D + lane * 4), k);
      unpack4(*reinterpret_cast<const uint32_t*>(v_cache + ((bh << a.log2_bs) + j) * D + lane * 4), v);
      const float s = warp_sum(qx.x * k[0] + qx.y * k[1] + qy.x * k[2] + qy.y * k[3]) * ks;
      const float mn = fmaxf(m, s);
      const float corr = mn == -INFINITY ? 1.f : exp2f(m - mn);
      const float p = mn == -INFINITY ? 0.f : exp2f(s - mn);
      m = mn;
      l = l * corr + p;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = o[i] * corr + p * vs * v[i];
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const uint2 r = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
  *reinterpret_cast<uint2*>(a.out + tok * a.out_ld + head * D + lane * 4) = r;
}

__global__ void __launch_bounds__(256) prefill_kernel(const Args a, const uint8_t* k_cache, const uint8_t* v_cache) {
  pdl_trigger();
  pdl_wait();
  const int seq = a.tile_seq[blockIdx.x];
  if (seq < 0) return;
  const int row0 = a.tile_row0[blockIdx.x];
  if (seq >= a.num_seqs || row0 < 0) {
    if (threadIdx.x == 0) record_error(a.err, kErrBounds);
    return;
  }
  const int q0 = a.cu_q[seq], n = a.cu_q[seq + 1] - q0, len = a.seq_lens[seq];
  for (int r = row0 + (threadIdx.x >> 5); r < min(row0 + 256, n * a.group); r += 8) {
    const int tok = r / a.group, g = r % a.group;
    const int klim = a.causal ? max(0, min(len, len - n + tok + 1)) : len;
    attend(a, k_cache, v_cache, seq, q0 + tok, blockIdx.y * a.group + g, klim, threadIdx.x & 31);
  }
}

}  // namespace fp8a

void paged_attention_fp8(const at::Tensor& q, const at::Tensor& k_cache,
                         const at::Tensor& v_cache, const at::Tensor& k_scale,
                         const at::Tensor& v_scale, at::Tensor& out,
                         const at::Tensor& block_tables, const at::Tensor& seq_lens,
                         const c10::optional<at::Tensor>& cu_q,
                         const c10::optional<at::Tensor>& tile_seq,
                         const c10::optional<at::Tensor>& tile_row0, int64_t group, double scale,
                         bool decode, bool causal, at::Tensor& err) {
  using namespace fp8a;
  const char* op = "paged_attention_fp8";
  check_fp8_cache(op, k_cache, v_cache, k_scale, v_scale);
  for (const at::Tensor* t : {&q, (const at::Tensor*)&out})
    TORCH_CHECK(t->is_cuda() && t->scalar_type() == at::kBFloat16 && t->dim() == 3 &&
                    t->size(2) == D && t->stride(2) == 1 && (t->size(1) <= 1 || t->stride(1) == D) &&
                    (t->size(0) <= 1 || t->stride(0) % 8 == 0) &&
                    reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                op, ": q and out are bf16 [T, Hq, 128], contiguous heads, 16-byte aligned rows");
  TORCH_CHECK(q.sizes() == out.sizes(), op, ": out has q's shape");
  TORCH_CHECK(group >= 1 && q.size(1) == group * k_cache.size(1), op, ": Hq = group * Hkv");
  const int64_t B = seq_lens.numel();
  TORCH_CHECK(block_tables.is_cuda() && block_tables.scalar_type() == at::kInt &&
                  block_tables.dim() == 2 && block_tables.size(0) >= B &&
                  (block_tables.size(1) <= 1 || block_tables.stride(1) == 1) &&
                  seq_lens.is_cuda() && seq_lens.scalar_type() == at::kInt &&
                  seq_lens.is_contiguous(),
              op, ": block_tables [B, W] and seq_lens [B] are int32");
  Args a;
  a.q = reinterpret_cast<const bf16*>(q.data_ptr());
  a.q_ld = q.stride(0);
  a.out = reinterpret_cast<bf16*>(out.data_ptr());
  a.out_ld = out.stride(0);
  a.k_scale = k_scale.data_ptr<float>();
  a.v_scale = v_scale.data_ptr<float>();
  a.tables = block_tables.data_ptr<int>();
  a.bt_stride = block_tables.stride(0);
  a.bt_width = block_tables.size(1);
  a.seq_lens = seq_lens.data_ptr<int>();
  a.cu_q = nullptr;
  a.tile_seq = a.tile_row0 = nullptr;
  a.hq = q.size(1);
  a.hkv = k_cache.size(1);
  a.group = group;
  a.log2_bs = k_cache.size(2) == 16 ? 4 : k_cache.size(2) == 32 ? 5 : 6;
  a.num_blocks = k_cache.size(0);
  a.num_seqs = B;
  a.causal = causal ? 1 : 0;
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  a.err = err.data_ptr<int>();
  // a row of 128 codes is 64 two-byte elements to the tensor map
  const uint64_t rows = k_cache.size(0) * k_cache.size(1) * k_cache.size(2);
  const CUtensorMap tk =
      make_tmap_bf16_2d(k_cache.data_ptr(), 64, rows, D, 64, SL, CU_TENSOR_MAP_SWIZZLE_128B);
  const CUtensorMap tv =
      make_tmap_bf16_2d(v_cache.data_ptr(), 64, rows, D, 64, SL, CU_TENSOR_MAP_SWIZZLE_128B);
  cudaStream_t st = at::cuda::getCurrentCUDAStream();
  if (decode) {
    TORCH_CHECK(q.size(0) >= B, op, ": one query token per sequence");
    if (B == 0) return;
    fp8_decode(a, tk, tv, q, st);
    return;
  }
  TORCH_CHECK(cu_q.has_value() && tile_seq.has_value() && tile_row0.has_value(), op,
              ": prefill needs cu_q and the work list (tile_seq, tile_row0)");
  for (const at::Tensor* t : {&*cu_q, &*tile_seq, &*tile_row0})
    TORCH_CHECK(t->is_cuda() && t->scalar_type() == at::kInt && t->is_contiguous(), op,
                ": cu_q and the work list are contiguous int32");
  TORCH_CHECK(cu_q->numel() >= B + 1 && tile_seq->numel() == tile_row0->numel(), op, ": sizes");
  if (B == 0 || tile_seq->numel() == 0) return;
  a.cu_q = cu_q->data_ptr<int>();
  a.tile_seq = tile_seq->data_ptr<int>();
  a.tile_row0 = tile_row0->data_ptr<int>();
  C10_CUDA_CHECK(launch_k(prefill_kernel, dim3(tile_seq->numel(), a.hkv), dim3(256), 0, st,
                          nullptr, 0, a, reinterpret_cast<const uint8_t*>(k_cache.data_ptr()),
                          reinterpret_cast<const uint8_t*>(v_cache.data_ptr())));
}

}  // namespace lb
