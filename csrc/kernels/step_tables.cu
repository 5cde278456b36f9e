// Block tables, slot map, positions and attention work list of one engine step, built on the
// device from the requests' lengths (sm_100a).
//
//   have_b  = ceil(c_b / BS)             blocks request b already has (c_b cached tokens)
//   need_b  = ceil((c_b + n_b) / BS)     blocks it has after this step (n_b new tokens)
//   start_b = sum_{a < b} (need_a - have_a)
//   table[row_b][j] = new_blocks[start_b + j - have_b]          have_b <= j < need_b
//   cu_q = exclusive sum of n;  token i of b: pos = c_b + i - cu_q[b],
//   slot = table[row_b][pos / BS] * BS + pos % BS
//   tiles: (b, R r) for r < ceil(n_b G / R), requests in order
//
// A few hundred kilobytes at most, so the cost is one launch and a chain of dependent loads
// (lengths -> scan -> table entry -> slot).  One launch does everything without talking between
// CTAs: each CTA repeats the three exclusive sums over the requests (shared memory, one warp
// shuffle scan per 256 requests; the lengths come from L2) and then fills its own share of
// tokens, table entries and tiles, finding the owner of an item by bisection in shared memory.
// A slot in a block that this step adds is taken from new_blocks, never from the table that
// another CTA is writing.  Table rows are copied in pieces of 128 entries per warp: with a warp per
// row, 40 rows of 1907 entries took 13.9 us.  Measured: 3.6 us for 256 requests of one token, 3.4 us
// for 40 chunks of up to 512 tokens behind 30,000; a launch that does nothing takes about 2.
#include <ATen/Functions.h>
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include "checks.h"
#include "common.cuh"

namespace lb {
namespace st {

constexpr int THREADS = 256;
constexpr int MAX_B = 4096;
constexpr int SEG = 128;          // table entries per warp step

struct Args {
  const int* ctx;
  const int* q;
  const int* rows;        // nullptr: request b is row b
  int* seq_tables;
  int64_t tab_stride;
  const int* new_blocks;
  int* block_tables;      // [B, W]
  int* seq_lens;
  int* cu_q;
  int* positions;
  int* slots;
  int* last_rows;
  int* tile_seq;
  int* tile_row0;
  int* num_new;
  int* err;
  int B, S, W, F, T, log2_bs, group, rows_per_tile, num_tiles, num_decode;
};

// Largest b with s[b] <= i (s non-decreasing, s[0] = 0, i < s[n]): empty requests are skipped.
__device__ __forceinline__ int owner(const int* s, int n, int i) {
  int lo = 0, hi = n;               // s[lo] <= i < s[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(THREADS) step_tables_kernel(const Args a) {
  extern __shared__ int sm[];
  int* sq = sm;                     // [B + 1] first token
  int* sn = sq + a.B + 1;           // [B + 1] first new block
  int* stl = sn + a.B + 1;          // [B + 1] first tile
  int* sc = stl + a.B + 1;          // [B] cached tokens
  __shared__ int warp_tot[3][THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_trigger();
  pdl_wait();
  const int bs = 1 << a.log2_bs;
  int base[3] = {0, 0, 0};
  bool bad = false;
  for (int b0 = 0; b0 < a.B; b0 += THREADS) {
    const int b = b0 + tid;
    int v[3] = {0, 0, 0}, c = 0;
    if (b < a.B) {
      c = a.ctx[b];
      int n = a.q[b];
      const int row = a.rows != nullptr ? a.rows[b] : b;
      // lengths or rows that the tables cannot hold: reported, the request counts as empty
      if (c < 0 || n < 0 || static_cast<unsigned>(row) >= static_cast<unsigned>(a.S) ||
          static_cast<long long>(c) + n > static_cast<long long>(a.W) * bs) {
        bad = true;
        c = n = 0;
      }
      v[0] = n;
      v[1] = ((c + n + bs - 1) >> a.log2_bs) - ((c + bs - 1) >> a.log2_bs);
      v[2] = b < a.num_decode ? 0 : static_cast<int>((static_cast<long long>(n) * a.group +
                                                      a.rows_per_tile - 1) / a.rows_per_tile);
      sc[b] = c;
    }
    int incl[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      incl[k] = v[k];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl[k], o);
        if (lane >= o) incl[k] += up;
      }
      if (lane == 31) warp_tot[k][warp] = incl[k];
    }
    __syncthreads();
    int tot[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      int before = 0, all = 0;
      for (int w = 0; w < THREADS / 32; ++w) {
        const int x = warp_tot[k][w];
        if (w < warp) before += x;
        all += x;
      }
      incl[k] += base[k] + before;
      tot[k] = all;
    }
    if (b < a.B) {
      sq[b + 1] = incl[0];
      sn[b + 1] = incl[1];
      stl[b + 1] = incl[2];
    }
    if (b0 == 0 && tid == 0) sq[0] = sn[0] = stl[0] = 0;
#pragma unroll
    for (int k = 0; k < 3; ++k) base[k] += tot[k];
    __syncthreads();
  }
  const int tokens = sq[a.B], fresh = sn[a.B], tiles = stl[a.B];
  if (blockIdx.x == 0) {
    if (tid == 0) {
      a.num_new[0] = fresh;
      a.cu_q[0] = 0;
      bad |= tokens > a.T || fresh > a.F;
    }
    for (int b = tid; b < a.B; b += THREADS) {
      const int n = sq[b + 1] - sq[b];
      a.cu_q[b + 1] = sq[b + 1];
      a.seq_lens[b] = sc[b] + n;
      a.last_rows[b] = n > 0 ? sq[b + 1] - 1 : -1;
    }
  }
  const int nthreads = gridDim.x * THREADS;
  const int gt = blockIdx.x * THREADS + tid;
  for (int i = gt; i < a.T; i += nthreads) {
    int pos = 0, slot = -1;
    if (i < tokens) {
      const int b = owner(sq, a.B, i);
      pos = sc[b] + i - sq[b];
      const int j = pos >> a.log2_bs;
      const int have = (sc[b] + bs - 1) >> a.log2_bs;
      int id = -1;
      if (j < have) {
        const int row = a.rows != nullptr ? a.rows[b] : b;
        id = a.seq_tables[row * a.tab_stride + j];
      } else if (sn[b] + j - have < a.F) {
        id = a.new_blocks[sn[b] + j - have];
      }
      if (id < 0 || id > (0x7fffffff >> a.log2_bs) - 1) bad = true;
      else slot = (id << a.log2_bs) + (pos & (bs - 1));
    }
    a.positions[i] = pos;
    a.slots[i] = slot;
  }
  // the batch's tables, SEG entries of one request per warp; new entries also go to the resident
  // table
  const int segs = (a.W + SEG - 1) / SEG;
  for (int i = gt >> 5; i < a.B * segs; i += nthreads >> 5) {
    const int b = i / segs, j0 = (i - b * segs) * SEG + lane;
    const int n = sq[b + 1] - sq[b];
    const int have = (sc[b] + bs - 1) >> a.log2_bs, need = (sc[b] + n + bs - 1) >> a.log2_bs;
    const int row = a.rows != nullptr ? a.rows[b] : b;
    int* src = a.seq_tables + (need > 0 ? row * a.tab_stride : 0);
    int* dst = a.block_tables + static_cast<int64_t>(b) * a.W;
    int id[SEG / 32];
#pragma unroll
    for (int k = 0; k < SEG / 32; ++k) {
      const int j = j0 + 32 * k, f = sn[b] + j - have;
      id[k] = j < have ? src[j] : j < need && f < a.F ? a.new_blocks[f] : 0;
    }
#pragma unroll
    for (int k = 0; k < SEG / 32; ++k) {
      const int j = j0 + 32 * k;
      if (j < a.W) dst[j] = id[k];
      if (j >= have && j < need && sn[b] + j - have < a.F) src[j] = id[k];
    }
  }
  for (int i = gt; i < a.num_tiles; i += nthreads) {
    int s = -1, r = 0;
    if (i < tiles) {
      s = owner(stl, a.B, i);
      r = (i - stl[s]) * a.rows_per_tile;
    }
    a.tile_seq[i] = s;
    a.tile_row0[i] = r;
  }
  if (bad) record_error(a.err, kErrBounds);
}

}  // namespace st

// Contiguous int32 view of `n` elements (or [r, n / r]) of a buffer.
static at::Tensor view_of(const at::Tensor& buf, int64_t offset, at::IntArrayRef sizes) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(
      c10::Storage(buf.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA), buf.dtype());
  impl->set_storage_offset(offset);
  impl->set_sizes_contiguous(sizes);
  return at::Tensor(std::move(impl));
}

std::vector<at::Tensor> step_tables(const at::Tensor& ctx_lens, const at::Tensor& q_lens,
                                    const c10::optional<at::Tensor>& rows, at::Tensor& seq_tables,
                                    const at::Tensor& new_blocks, int64_t num_tokens,
                                    int64_t block_size, int64_t group, int64_t rows_per_tile,
                                    int64_t num_decode, at::Tensor& err) {
  using namespace st;
  const int64_t B = ctx_lens.numel(), T = num_tokens;
  for (const at::Tensor* t : {&ctx_lens, &q_lens, &new_blocks})
    TORCH_CHECK(t->is_cuda() && t->scalar_type() == at::kInt && t->is_contiguous(),
                "step_tables: lengths and new_blocks are contiguous int32 CUDA tensors");
  TORCH_CHECK(seq_tables.is_cuda() && seq_tables.scalar_type() == at::kInt &&
                  seq_tables.dim() == 2 && (seq_tables.size(1) <= 1 || seq_tables.stride(1) == 1),
              "step_tables: seq_tables [S, W] int32, contiguous rows");
  const bool has_rows = rows.has_value() && rows->defined();
  check_same_device("step_tables", ctx_lens, {&q_lens, has_rows ? &*rows : nullptr, &seq_tables,
                                              &new_blocks, &err});
  const c10::cuda::CUDAGuard guard(ctx_lens.device());
  const int64_t W = seq_tables.size(1);
  if (has_rows)
    TORCH_CHECK(rows->is_cuda() && rows->scalar_type() == at::kInt && rows->is_contiguous() &&
                    rows->numel() == B,
                "step_tables: rows [B] int32");
  TORCH_CHECK(B >= 1 && B <= MAX_B && q_lens.numel() == B, "step_tables: 1 to ", MAX_B,
              " requests");
  TORCH_CHECK(block_size >= 1 && block_size <= 1024 && (block_size & (block_size - 1)) == 0,
              "step_tables: power-of-two block size");
  TORCH_CHECK(group >= 1 && rows_per_tile >= 1 && T >= 0, "step_tables: group, rows_per_tile");
  TORCH_CHECK(W >= 1 && W * block_size < (int64_t(1) << 31) && T * group < (int64_t(1) << 31) &&
                  B * W < (int64_t(1) << 31),
              "step_tables: table width or token count");
  const int64_t tiles = T * group / rows_per_tile + B;
  // one allocation, every output on a 16-byte boundary
  int64_t used = 0;
  auto place = [&](int64_t n) {
    const int64_t at = used;
    used += (n + 3) / 4 * 4;
    return at;
  };
  const int64_t o_tab = place(B * W), o_len = place(B), o_cu = place(B + 1), o_pos = place(T),
                o_slot = place(T), o_last = place(B), o_ts = place(tiles), o_tr = place(tiles),
                o_new = place(1);
  at::Tensor buf = at::empty({used}, ctx_lens.options());
  int* p = buf.data_ptr<int>();
  Args a;
  a.ctx = ctx_lens.data_ptr<int>();
  a.q = q_lens.data_ptr<int>();
  a.rows = has_rows ? rows->data_ptr<int>() : nullptr;
  a.seq_tables = seq_tables.data_ptr<int>();
  a.tab_stride = seq_tables.stride(0);
  a.new_blocks = new_blocks.data_ptr<int>();
  a.block_tables = p + o_tab;
  a.seq_lens = p + o_len;
  a.cu_q = p + o_cu;
  a.positions = p + o_pos;
  a.slots = p + o_slot;
  a.last_rows = p + o_last;
  a.tile_seq = p + o_ts;
  a.tile_row0 = p + o_tr;
  a.num_new = p + o_new;
  a.err = err.data_ptr<int>();
  a.B = B;
  a.S = seq_tables.size(0);
  a.W = W;
  a.F = new_blocks.numel();
  a.T = T;
  a.log2_bs = 0;
  while ((1 << a.log2_bs) < block_size) ++a.log2_bs;
  a.group = group;
  a.rows_per_tile = rows_per_tile;
  a.num_tiles = tiles;
  a.num_decode = num_decode;
  const int64_t items = std::max<int64_t>({B * ((W + SEG - 1) / SEG) * 32, T, tiles});
  const int grid = static_cast<int>(std::min<int64_t>(148, (items + THREADS - 1) / THREADS));
  const size_t smem = (4 * B + 3) * sizeof(int);
  if (smem > 48 * 1024)
    C10_CUDA_CHECK(cudaFuncSetAttribute(step_tables_kernel,
                                        cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        static_cast<int>((4 * MAX_B + 3) * sizeof(int))));
  C10_CUDA_CHECK(launch_k(step_tables_kernel, dim3(grid), dim3(THREADS), smem,
                          at::cuda::getCurrentCUDAStream(), nullptr, 0, a));
  return {view_of(buf, o_tab, {B, W}), view_of(buf, o_len, {B}), view_of(buf, o_cu, {B + 1}),
          view_of(buf, o_pos, {T}), view_of(buf, o_slot, {T}), view_of(buf, o_last, {B}),
          view_of(buf, o_ts, {tiles}), view_of(buf, o_tr, {tiles}), view_of(buf, o_new, {1})};
}

}  // namespace lb
