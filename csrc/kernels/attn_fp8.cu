// Paged attention over the 8-bit KV cache (sm_100a).
//
//   s_j = scale * ks_{b(j)} * (q . k8_j),  p_j = exp(s_j - max s),
//   o   = sum_j p_j vs_{b(j)} v8_j / sum_j p_j
//
// Argument checks and the choice of kernel: attn_fp8_rows.cu for one query token per sequence and
// for work lists of few rows an item, attn_fp8_prefill.cu (tcgen05) for the rest.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include "attn_fp8.cuh"
#include "checks.h"

namespace lb {

void check_fp8_cache(const char* op, const at::Tensor& k_cache, const at::Tensor& v_cache,
                     const at::Tensor& k_scale, const at::Tensor& v_scale);

// Returns the number of kernels launched.
int64_t paged_attention_fp8(const at::Tensor& q, const at::Tensor& k_cache,
                            const at::Tensor& v_cache, const at::Tensor& k_scale,
                            const at::Tensor& v_scale, at::Tensor& out,
                            const at::Tensor& block_tables, const at::Tensor& seq_lens,
                            const c10::optional<at::Tensor>& cu_q,
                            const c10::optional<at::Tensor>& tile_seq,
                            const c10::optional<at::Tensor>& tile_row0, int64_t group, double scale,
                            bool decode, bool causal, int64_t item_rows, at::Tensor& err) {
  using namespace fp8a;
  const char* op = "paged_attention_fp8";
  check_fp8_cache(op, k_cache, v_cache, k_scale, v_scale);
  const bool list = !decode && cu_q.has_value() && tile_seq.has_value() && tile_row0.has_value();
  TORCH_CHECK(decode || list, op, ": prefill needs cu_q and the work list (tile_seq, tile_row0)");
  check_same_device(op, k_cache, {&q, &out, &block_tables, &seq_lens, &err, list ? &*cu_q : nullptr,
                                  list ? &*tile_seq : nullptr, list ? &*tile_row0 : nullptr});
  const c10::cuda::CUDAGuard guard(k_cache.device());
  for (const at::Tensor* t : {&q, (const at::Tensor*)&out})
    TORCH_CHECK(t->is_cuda() && t->scalar_type() == at::kBFloat16 && t->dim() == 3 &&
                    t->size(2) == D && t->stride(2) == 1 && (t->size(1) <= 1 || t->stride(1) == D) &&
                    (t->size(0) <= 1 || t->stride(0) % 8 == 0) &&
                    reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                op, ": q and out are bf16 [T, Hq, 128], contiguous heads, 16-byte aligned rows");
  TORCH_CHECK(q.sizes() == out.sizes(), op, ": out has q's shape");
  TORCH_CHECK(group >= 1 && q.size(1) == group * k_cache.size(1), op, ": Hq = group * Hkv");
  TORCH_CHECK(q.size(0) * group < (int64_t(1) << 31) - 256, op, ": query rows exceed int32");
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
  a.tokens = static_cast<int>(q.size(0));
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
    if (B == 0) return 0;
    TORCH_CHECK(fp8_rows_fits(a, false), op,
                ": at most 4096 sequences, and 2^31 / 32 keys x KV heads in their tables");
    fp8_rows(a, false, group, tk, tv, q, st);
    return 2;
  }
  for (const at::Tensor* t : {&*cu_q, &*tile_seq, &*tile_row0})
    TORCH_CHECK(t->is_cuda() && t->scalar_type() == at::kInt && t->is_contiguous(), op,
                ": cu_q and the work list are contiguous int32");
  TORCH_CHECK(cu_q->numel() >= B + 1 && tile_seq->numel() == tile_row0->numel(), op, ": sizes");
  if (B == 0 || tile_seq->numel() == 0) return 0;
  a.cu_q = cu_q->data_ptr<int>();
  a.tile_seq = tile_seq->data_ptr<int>();
  a.tile_row0 = tile_row0->data_ptr<int>();
  a.num_tiles = tile_seq->numel();
  // At most FEW_ROWS query rows per item (verification of a few tokens, tails of prompts): 256-row tiles
  // would be mostly padding.  rows / tcgen05 kernel, us: 32 rows 64 x 4000 keys 193 / 311, 32 x 1280
  // 48 / 58; 48 rows 32 x 1280 62 / 58; 64 rows 79 / 59.  The caller says how many rows its longest item
  // has; a full item on the first kernel reads its keys 16 times (a 2048-token chunk over 16k beside 255
  // decodes 2999 us instead of 675).  Else the mean decides, over all of q and all entries.
  constexpr int64_t FEW_ROWS = 32;
  const int64_t rows_of_item =
      item_rows > 0 ? item_rows : (q.size(0) * group + a.num_tiles - 1) / a.num_tiles;
  if (rows_of_item <= FEW_ROWS && fp8_rows_fits(a, true)) {
    fp8_rows(a, true, rows_of_item, tk, tv, q, st);
    return 2;
  }
  fp8_prefill(a, tk, tv, st);
  return 1;
}

}  // namespace lb
