// TORCH_LIBRARY binding of libtrianglemix_hip.so, in the style the reference registers its own
// ROCm ops (csrc/rocm/torch_bindings.cpp:14-57, csrc/rocm/ops.h:17-26, csrc/core/registration.h:13-27):
// schema strings with `Tensor!` for mutated outputs, implementations on the CUDA dispatch key (HIP
// tensors dispatch there), outputs preallocated by the Python caller as vllm/_custom_ops.py:153-196
// does.  Tensors are unpacked to the pointers, strides and sizes of the C ABI; the work is enqueued
// on the current stream of the tensors' device; nothing synchronises with the host.
//
// Built as _trianglemix_C.so (plain C++, no device code) and loaded with
// torch.ops.load_library(); the ops then live under torch.ops._trianglemix_C.
#include <ATen/ops/empty.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <torch/library.h>

#include <optional>
#include <vector>

#include "trianglemix_hip.h"

namespace {

using at::Tensor;

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TMX_F32;
    case at::kBFloat16: return TMX_BF16;
    case at::kHalf: return TMX_F16;
    default: TORCH_CHECK(false, "trianglemix: unsupported dtype ", t.scalar_type());
  }
}

void check(int code) { TORCH_CHECK(code == TMX_OK, "trianglemix: ", tmx_last_error()); }

// PyTorch-ROCm presents HIP devices under the "cuda" device type; these are its guard and stream types for them.
using DeviceGuard = c10::hip::HIPGuardMasqueradingAsCUDA;
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

int32_t* i32(const Tensor& t) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous(), "trianglemix: index tensors must be contiguous int32");
  return t.data_ptr<int32_t>();
}

int32_t* i32_opt(const std::optional<Tensor>& t) { return t.has_value() ? i32(*t) : nullptr; }

// The eight index buffers travel as one list: row_ptr, col_idx, qb_meta, part_ptr, items, split_qb, totals, scratch.
void fill_index(tmx_index_t& ix, const std::vector<Tensor>& b, const std::optional<Tensor>& tile_pages,
                const std::optional<Tensor>& pages_block_table, int64_t page_size, int64_t si, int64_t sl,
                int64_t last, int64_t block_m, int64_t block_n, int64_t mode, int64_t tri_min_len,
                int64_t chunk_tiles, int64_t batch, const std::optional<Tensor>& full_lens = std::nullopt,
                const std::optional<Tensor>& full_lens_cpu = std::nullopt, int64_t dense_rows_from = 0) {
  TORCH_CHECK(b.size() == 8, "trianglemix: the index is a list of 8 tensors");
  ix = tmx_index_t{};
  ix.row_ptr = i32(b[0]);
  ix.col_idx = i32(b[1]);
  ix.qb_meta = i32(b[2]);
  ix.part_ptr = i32(b[3]);
  ix.items = i32(b[4]);
  ix.split_qb = i32(b[5]);
  ix.totals = i32(b[6]);
  ix.scratch = i32(b[7]);
  ix.cap_qblocks = b[0].numel() - 1;
  TORCH_CHECK(b[7].numel() >= TMX_INDEX_SCRATCH_INTS(batch, ix.cap_qblocks),
              "trianglemix: the index's scratch tensor has ", b[7].numel(), " entries, ",
              TMX_INDEX_SCRATCH_INTS(batch, ix.cap_qblocks), " are needed (batch + 1 + 2 (R + 1) + 8 (R / 1024 + 1))");
  ix.cap_nnz = b[1].numel();
  ix.cap_items = b[4].numel() / 8;
  ix.cap_split = b[5].numel();
  ix.block_m = (int32_t)block_m;
  ix.block_n = (int32_t)block_n;
  ix.mode = (int32_t)mode;
  ix.chunk_tiles = (int32_t)chunk_tiles;
  ix.si = (int32_t)si;
  ix.sl = (int32_t)sl;
  ix.last = (int32_t)last;
  ix.batch = (int32_t)batch;
  ix.tri_min_len = (int32_t)tri_min_len;
  if (tile_pages.has_value() && pages_block_table.has_value()) {
    ix.tile_pages = i32(*tile_pages);
    TORCH_CHECK(pages_block_table->scalar_type() == at::kInt && pages_block_table->stride(1) == 1,
                "trianglemix: block_table must be int32 with contiguous rows");
    ix.pages_block_table = pages_block_table->data_ptr<int32_t>();
    ix.pages_block_table_stride = pages_block_table->stride(0);
    ix.pages_page_size = (int32_t)page_size;
  }
  ix.full_lens = i32_opt(full_lens);
  ix.full_lens_host = i32_opt(full_lens_cpu);
  ix.dense_rows_from = (int32_t)dense_rows_from;
}

// Exact buffer sizes from the host copies of the batch: [R, nnz, items, partials, split q-blocks, max tiles].
std::vector<int64_t> index_sizes(const Tensor& cu_seqlens_q_cpu, const Tensor& seq_lens_cpu, int64_t si, int64_t sl,
                                 int64_t last, int64_t block_m, int64_t block_n, int64_t mode, int64_t tri_min_len,
                                 int64_t chunk_tiles, const std::optional<Tensor>& full_lens_cpu, int64_t dense_rows_from) {
  TORCH_CHECK(cu_seqlens_q_cpu.is_cpu() && seq_lens_cpu.is_cpu() && (!full_lens_cpu.has_value() || full_lens_cpu->is_cpu()),
              "trianglemix: host tensors expected");
  tmx_index_sizes_t sz;
  check(tmx_index_sizes_without_dense(i32(cu_seqlens_q_cpu), i32(seq_lens_cpu), i32_opt(full_lens_cpu), (int)seq_lens_cpu.numel(),
                                      (int)si, (int)sl, (int)last, (int)block_m, (int)block_n, (int)mode, (int)tri_min_len,
                                      (int)chunk_tiles, (int)dense_rows_from, &sz));
  return {sz.num_qblocks, sz.nnz_tiles, sz.num_items, sz.num_partials, sz.num_split_qblocks, sz.max_tiles_per_qblock};
}

// Piece length advice for a batch and a head grouping (host only).
int64_t suggest_chunk_tiles(const Tensor& cu_seqlens_q_cpu, const Tensor& seq_lens_cpu, int64_t si, int64_t sl,
                            int64_t last, int64_t block_m, int64_t block_n, int64_t mode, int64_t tri_min_len,
                            int64_t units_per_item, int64_t num_cus, const std::optional<Tensor>& full_lens_cpu) {
  TORCH_CHECK(cu_seqlens_q_cpu.is_cpu() && seq_lens_cpu.is_cpu(), "trianglemix: host tensors expected");
  int out = 0;
  check(tmx_suggest_chunk_tiles(i32(cu_seqlens_q_cpu), i32(seq_lens_cpu), i32_opt(full_lens_cpu),
                                (int)seq_lens_cpu.numel(), (int)si, (int)sl, (int)last, (int)block_m, (int)block_n,
                                (int)mode, (int)tri_min_len, (int)units_per_item, (int)num_cus, &out));
  return out;
}

void build_block_index(std::vector<Tensor> index, const std::optional<Tensor>& tile_pages, const Tensor& cu_seqlens_q,
                       const Tensor& seq_lens, const Tensor& cu_seqlens_q_cpu, const Tensor& seq_lens_cpu,
                       const std::optional<Tensor>& block_table, int64_t page_size, int64_t si, int64_t sl,
                       int64_t last, int64_t block_m, int64_t block_n, int64_t mode, int64_t tri_min_len,
                       int64_t chunk_tiles, const std::optional<Tensor>& full_lens,
                       const std::optional<Tensor>& full_lens_cpu, int64_t dense_rows_from) {
  const DeviceGuard guard(cu_seqlens_q.device());
  tmx_index_t ix;
  fill_index(ix, index, tile_pages, block_table, page_size, si, sl, last, block_m, block_n, mode, tri_min_len,
             chunk_tiles, seq_lens.numel(), full_lens, full_lens_cpu, dense_rows_from);
  check(tmx_build_block_index(&ix, i32(cu_seqlens_q), i32(seq_lens), i32(cu_seqlens_q_cpu), i32(seq_lens_cpu),
                              stream_of(cu_seqlens_q)));
}

// Every tensor that reaches the library as a device pointer must live on the GPU of `ref`.
void on_gpu(const Tensor& t, const Tensor& ref, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == ref.device(), "trianglemix: ", name, " must be on the HIP device of the query");
}
void on_gpu(const std::optional<Tensor>& t, const Tensor& ref, const char* name) {
  if (t.has_value()) on_gpu(*t, ref, name);
}

void attention(Tensor& out, const Tensor& query, const Tensor& key_cache, const Tensor& value_cache,
               const std::optional<Tensor>& block_table, const Tensor& cu_seqlens_q, const Tensor& seq_lens,
               const std::optional<Tensor>& cu_seqlens_k, std::vector<Tensor> index,
               const std::optional<Tensor>& tile_pages, const std::optional<Tensor>& partial_o,
               const std::optional<Tensor>& partial_ml, const std::optional<Tensor>& bias, double scale, int64_t si,
               int64_t sl, int64_t last, int64_t mode, int64_t tri_min_len, int64_t chunk_tiles, int64_t num_items,
               int64_t num_partials, int64_t num_split_qblocks, const std::optional<Tensor>& full_lens,
               int64_t flags, int64_t nnz_tiles, const std::optional<Tensor>& k_new, const std::optional<Tensor>& v_new,
               const std::optional<Tensor>& cache_slots, double k_scale, double v_scale, int64_t index_block_m,
               int64_t index_block_n, const std::optional<Tensor>& kv_stage, int64_t index_dense_rows_from) {
  TORCH_CHECK(query.is_cuda(), "trianglemix: query must be on a HIP device (there is no CPU path)");
  const DeviceGuard guard(query.device());
  TORCH_CHECK(query.dim() == 3 && out.dim() == 3 && query.sizes() == out.sizes(), "trianglemix: query / out must both be [T, H, D]");
  const bool paged = block_table.has_value();
  TORCH_CHECK(key_cache.dim() == (paged ? 4 : 3), "trianglemix: K/V must be [blocks, page, Hkv, D] (paged) or [rows, Hkv, D]");
  on_gpu(out, query, "out");
  on_gpu(key_cache, query, "key_cache");
  on_gpu(value_cache, query, "value_cache");
  on_gpu(cu_seqlens_q, query, "cu_seqlens_q");
  on_gpu(seq_lens, query, "seq_lens");
  on_gpu(block_table, query, "block_table");
  on_gpu(cu_seqlens_k, query, "cu_seqlens_k");
  on_gpu(tile_pages, query, "tile_pages");
  on_gpu(partial_o, query, "partial_o");
  on_gpu(partial_ml, query, "partial_ml");
  on_gpu(bias, query, "bias");
  on_gpu(full_lens, query, "full_lens");
  on_gpu(k_new, query, "k_new");
  on_gpu(v_new, query, "v_new");
  on_gpu(cache_slots, query, "cache_slots");
  for (const Tensor& t : index) on_gpu(t, query, "index");
  const bool fp8 = key_cache.element_size() == 1;  // uint8 / float8_e4m3fn: an fp8 cache read in place
  TORCH_CHECK(fp8 || (key_cache.scalar_type() == query.scalar_type() && value_cache.scalar_type() == query.scalar_type()),
              "trianglemix: q, k, v must share a dtype of bfloat16 or float16 (or K/V be an fp8 cache)");
  TORCH_CHECK(!fp8 || (paged && !bias.has_value() && query.size(2) == 128 && value_cache.element_size() == 1),
              "trianglemix: an fp8 K/V cache is read in place only in the paged layout, with head size 128 and no bias");
  TORCH_CHECK(key_cache.sizes() == value_cache.sizes() && key_cache.strides() == value_cache.strides(),
              "trianglemix: k and v must have the same shape and strides");
  TORCH_CHECK(query.stride(2) == 1 && out.stride(2) == 1 && key_cache.stride(-1) == 1,
              "trianglemix: the head dimension must be contiguous");
  TORCH_CHECK(key_cache.size(-1) == query.size(2), "trianglemix: k/v head size differs from q");
  tmx_index_t ix;
  const int64_t hkv = key_cache.size(paged ? 2 : 1);
  // the geometry the index was built with (0: the kernel's own; the library rejects any other)
  const int64_t block_m = index_block_m > 0 ? index_block_m : tmx_attention_block_m((int)query.size(1), (int)hkv);
  fill_index(ix, index, tile_pages, block_table, paged ? key_cache.size(1) : 0, si, sl, last, block_m,
             index_block_n > 0 ? index_block_n : tmx_attention_block_n(), mode, tri_min_len, chunk_tiles, seq_lens.numel(),
             full_lens, std::nullopt, index_dense_rows_from);
  tmx_attention_args_t a{};
  a.struct_size = sizeof(a);
  a.io_dtype = dtype_code(query);
  a.out_dtype = dtype_code(out);
  a.mode = (int32_t)mode;
  a.si = (int32_t)si;
  a.sl = (int32_t)sl;
  a.last = (int32_t)last;
  a.scale = (float)scale;
  a.batch = (int32_t)seq_lens.numel();
  a.num_heads = (int32_t)query.size(1);
  a.num_kv_heads = (int32_t)hkv;
  a.head_dim = (int32_t)query.size(2);
  a.total_q = (int32_t)query.size(0);
  a.out = out.data_ptr();
  a.out_stride_t = out.stride(0);
  a.out_stride_h = out.stride(1);
  a.q = query.data_ptr();
  a.q_stride_t = query.stride(0);
  a.q_stride_h = query.stride(1);
  a.k = key_cache.data_ptr();
  a.v = value_cache.data_ptr();
  if (paged) {
    a.kv_stride_page = key_cache.stride(0);
    a.kv_stride_t = key_cache.stride(1);
    a.kv_stride_h = key_cache.stride(2);
    TORCH_CHECK(block_table->scalar_type() == at::kInt && block_table->dim() == 2 && block_table->stride(1) == 1 &&
                    block_table->size(0) >= seq_lens.numel(),
                "trianglemix: block_table must be int32 [B, max_blocks] with contiguous rows that cover the batch");
    a.block_table = block_table->data_ptr<int32_t>();
    a.block_table_stride = block_table->stride(0);
    a.page_size = (int32_t)key_cache.size(1);
  } else {
    TORCH_CHECK(cu_seqlens_k.has_value(), "trianglemix: contiguous K/V needs cu_seqlens_k");
    a.kv_stride_t = key_cache.stride(0);
    a.kv_stride_h = key_cache.stride(1);
    a.cu_seqlens_k = i32(*cu_seqlens_k);
  }
  if (fp8) {
    a.kv_dtype = TMX_FP8_E4M3;
    a.k_scale = (float)k_scale;
    a.v_scale = (float)v_scale;
  } else {
    a.k_scale = a.v_scale = 1.0f;
  }
  TORCH_CHECK(k_new.has_value() == v_new.has_value(), "trianglemix: k_new and v_new go together");
  if (k_new.has_value()) {
    TORCH_CHECK(paged && !fp8, "trianglemix: k_new / v_new need a 16-bit paged cache");
    TORCH_CHECK(k_new->dim() == 3 && k_new->sizes() == v_new->sizes() && k_new->strides() == v_new->strides() &&
                    k_new->stride(2) == 1 && k_new->scalar_type() == query.scalar_type() &&
                    v_new->scalar_type() == query.scalar_type() && k_new->size(0) >= query.size(0) &&
                    k_new->size(1) == hkv && k_new->size(2) == query.size(2),
                "trianglemix: k_new / v_new must be [T, Hkv, D] rows of the q dtype with equal strides");
    a.k_new = k_new->data_ptr();
    a.v_new = v_new->data_ptr();
    a.new_stride_t = k_new->stride(0);
    a.new_stride_h = k_new->stride(1);
  }
  if (cache_slots.has_value()) {
    TORCH_CHECK(k_new.has_value() && cache_slots->scalar_type() == at::kLong && cache_slots->is_contiguous() &&
                    cache_slots->numel() >= query.size(0),
                "trianglemix: cache_slots must be contiguous int64 [T] and comes with k_new / v_new");
    a.cache_slots = cache_slots->data_ptr<int64_t>();
  }
  a.cu_seqlens_q = i32(cu_seqlens_q);
  a.seq_lens = i32(seq_lens);
  if (bias.has_value()) {
    a.bias = bias->data_ptr();
    a.bias_dtype = dtype_code(*bias);
    TORCH_CHECK(bias->dim() == 2 || bias->dim() == 4, "trianglemix: bias must be [rows, cols] or [1|B, 1|H, rows, cols]");
    const int64_t d0 = bias->dim() - 2;
    TORCH_CHECK(bias->stride(d0 + 1) == 1, "trianglemix: bias rows must be contiguous");
    a.bias_stride = bias->stride(d0);
    a.bias_rows = (int32_t)bias->size(d0);
    a.bias_cols = (int32_t)bias->size(d0 + 1);
    if (bias->dim() == 4) {
      TORCH_CHECK((bias->size(0) == 1 || bias->size(0) == seq_lens.numel()) && (bias->size(1) == 1 || bias->size(1) == query.size(1)),
                  "trianglemix: a 4-D bias is [1|batch, 1|heads, rows, cols]");
      a.bias_stride_b = bias->size(0) > 1 ? bias->stride(0) : 0;
      a.bias_stride_h = bias->size(1) > 1 ? bias->stride(1) : 0;
    }
  }
  a.index = &ix;
  a.num_items = num_items;
  a.num_partials = num_partials;
  a.num_split_qblocks = num_split_qblocks;
  a.nnz_tiles = nnz_tiles;  // 0: unknown (the library then falls back to the capacity of col_idx)
  if (num_partials > 0) {
    const int64_t need = num_partials * query.size(1) * block_m;
    TORCH_CHECK(partial_o.has_value() && partial_ml.has_value() && partial_o->scalar_type() == at::kFloat &&
                    partial_ml->scalar_type() == at::kFloat && partial_o->is_contiguous() && partial_ml->is_contiguous() &&
                    partial_o->numel() >= need * query.size(2) && partial_ml->numel() >= need * 2,
                "trianglemix: attention workspace too small for this index");
  }
  a.partial_o = partial_o.has_value() ? partial_o->data_ptr<float>() : nullptr;
  a.partial_ml = partial_ml.has_value() ? partial_ml->data_ptr<float>() : nullptr;
  a.flags = (uint32_t)flags;
  if (kv_stage.has_value()) {
    // staging area of the dense causal kernel: [2][rows][Hkv][128] 16-bit values
    on_gpu(*kv_stage, query, "kv_stage");
    TORCH_CHECK(kv_stage->dim() == 4 && kv_stage->size(0) == 2 && kv_stage->size(2) == hkv && kv_stage->size(3) == 128 &&
                    kv_stage->element_size() == 2 && kv_stage->is_contiguous(),
                "trianglemix: kv_stage must be a contiguous 16-bit [2, rows, Hkv, 128] tensor");
    a.kv_stage = kv_stage->data_ptr();
    a.kv_stage_rows = kv_stage->size(1);
  }
  check(tmx_attention(&a, stream_of(query)));
}

// A step of one-row requests with a launch that depends on the batch size alone (tmx_decode_attention): what the
// backend calls for uniform single-token decode steps, and what replays under a graph.
void decode_attention(Tensor& out, const Tensor& query, const Tensor& key_cache, const Tensor& value_cache,
                      const Tensor& block_table, const Tensor& seq_lens, Tensor& partial_o, Tensor& partial_ml,
                      double scale, const std::optional<Tensor>& k_new, const std::optional<Tensor>& v_new,
                      const std::optional<Tensor>& cache_slots, double k_scale, double v_scale) {
  TORCH_CHECK(query.is_cuda(), "trianglemix: query must be on a HIP device (there is no CPU path)");
  const DeviceGuard guard(query.device());
  TORCH_CHECK(query.dim() == 3 && out.dim() == 3 && query.sizes() == out.sizes() && query.stride(2) == 1 && out.stride(2) == 1,
              "trianglemix: query / out must both be [B, H, D] with a contiguous head dimension");
  TORCH_CHECK(key_cache.dim() == 4 && key_cache.sizes() == value_cache.sizes() && key_cache.strides() == value_cache.strides() &&
                  key_cache.stride(3) == 1 && key_cache.size(3) == query.size(2),
              "trianglemix: paged K/V: caches [num_blocks, page_size, Hkv, D] with equal strides");
  on_gpu(out, query, "out");
  on_gpu(key_cache, query, "key_cache");
  on_gpu(value_cache, query, "value_cache");
  on_gpu(block_table, query, "block_table");
  on_gpu(seq_lens, query, "seq_lens");
  on_gpu(partial_o, query, "partial_o");
  on_gpu(partial_ml, query, "partial_ml");
  on_gpu(k_new, query, "k_new");
  on_gpu(v_new, query, "v_new");
  on_gpu(cache_slots, query, "cache_slots");
  const int64_t B = query.size(0);
  TORCH_CHECK(seq_lens.scalar_type() == at::kInt && seq_lens.is_contiguous() && seq_lens.numel() >= B,
              "trianglemix: seq_lens must be contiguous int32 [B]");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.stride(1) == 1 &&
                  block_table.size(0) >= B,
              "trianglemix: block_table must be int32 [B, max_blocks] with contiguous rows that cover the batch");
  const bool fp8 = key_cache.element_size() == 1;
  TORCH_CHECK(fp8 ? value_cache.element_size() == 1
                  : (key_cache.scalar_type() == query.scalar_type() && value_cache.scalar_type() == query.scalar_type()),
              "trianglemix: q, k, v must share a dtype of bfloat16 or float16 (or K/V be an fp8 cache)");
  TORCH_CHECK(partial_o.scalar_type() == at::kFloat && partial_ml.scalar_type() == at::kFloat && partial_o.is_contiguous() &&
                  partial_ml.is_contiguous(),
              "trianglemix: the decode work area is two contiguous float32 tensors");
  tmx_decode_args_t a{};
  a.struct_size = sizeof(a);
  a.io_dtype = dtype_code(query);
  a.out_dtype = dtype_code(out);
  a.scale = (float)scale;
  a.batch = (int32_t)B;
  a.num_heads = (int32_t)query.size(1);
  a.num_kv_heads = (int32_t)key_cache.size(2);
  a.head_dim = (int32_t)query.size(2);
  a.out = out.data_ptr();
  a.out_stride_t = out.stride(0);
  a.out_stride_h = out.stride(1);
  a.q = query.data_ptr();
  a.q_stride_t = query.stride(0);
  a.q_stride_h = query.stride(1);
  a.k = key_cache.data_ptr();
  a.v = value_cache.data_ptr();
  a.kv_stride_page = key_cache.stride(0);
  a.kv_stride_t = key_cache.stride(1);
  a.kv_stride_h = key_cache.stride(2);
  a.block_table = block_table.data_ptr<int32_t>();
  a.block_table_stride = block_table.stride(0);
  a.page_size = (int32_t)key_cache.size(1);
  a.kv_dtype = fp8 ? TMX_FP8_E4M3 : 0;
  a.k_scale = fp8 ? (float)k_scale : 1.0f;
  a.v_scale = fp8 ? (float)v_scale : 1.0f;
  TORCH_CHECK(k_new.has_value() == v_new.has_value(), "trianglemix: k_new and v_new go together");
  if (k_new.has_value()) {
    TORCH_CHECK(k_new->dim() == 3 && k_new->sizes() == v_new->sizes() && k_new->strides() == v_new->strides() &&
                    k_new->stride(2) == 1 && k_new->scalar_type() == query.scalar_type() &&
                    v_new->scalar_type() == query.scalar_type() && k_new->size(0) >= B &&
                    k_new->size(1) == key_cache.size(2) && k_new->size(2) == query.size(2),
                "trianglemix: k_new / v_new must be [B, Hkv, D] rows of the q dtype with equal strides");
    a.k_new = k_new->data_ptr();
    a.v_new = v_new->data_ptr();
    a.new_stride_t = k_new->stride(0);
    a.new_stride_h = k_new->stride(1);
  }
  if (cache_slots.has_value()) {
    TORCH_CHECK(k_new.has_value() && cache_slots->scalar_type() == at::kLong && cache_slots->is_contiguous() &&
                    cache_slots->numel() >= B,
                "trianglemix: cache_slots must be contiguous int64 [B] and comes with k_new / v_new");
    a.cache_slots = cache_slots->data_ptr<int64_t>();
  }
  a.seq_lens = seq_lens.data_ptr<int32_t>();
  a.partial_o = partial_o.data_ptr<float>();
  a.partial_ml = partial_ml.data_ptr<float>();
  a.workspace_rows = std::min<int64_t>(partial_o.numel() / query.size(2), partial_ml.numel() / 2);
  check(tmx_decode_attention(&a, stream_of(query)));
}

void reshape_and_cache(const Tensor& key, const Tensor& value, Tensor& key_cache, Tensor& value_cache,
                       const Tensor& slot_mapping) {
  const DeviceGuard guard(key.device());
  TORCH_CHECK(slot_mapping.scalar_type() == at::kLong && slot_mapping.is_contiguous(),
              "trianglemix: slot_mapping must be contiguous int64");
  const int64_t n = std::min<int64_t>(slot_mapping.numel(), key.size(0));
  check(tmx_reshape_and_cache(key.data_ptr(), value.data_ptr(), key.stride(0), key.stride(1), key_cache.data_ptr(),
                              value_cache.data_ptr(), key_cache.stride(0), key_cache.stride(1), key_cache.stride(2),
                              slot_mapping.data_ptr<int64_t>(), (int32_t)n, (int32_t)key.size(1), (int32_t)key.size(2),
                              (int32_t)key_cache.size(1), dtype_code(key), stream_of(key)));
}

// fp8 (e4m3fn) caches arrive as uint8 or float8_e4m3fn tensors; strides of a one-byte type are bytes.
void* fp8_ptr(const Tensor& t) {
  TORCH_CHECK(t.element_size() == 1, "trianglemix: an fp8 cache is a one-byte tensor (uint8 / float8_e4m3fn)");
  return t.data_ptr();
}

void reshape_and_cache_fp8(const Tensor& key, const Tensor& value, Tensor& key_cache, Tensor& value_cache,
                           const Tensor& slot_mapping, double k_scale, double v_scale) {
  const DeviceGuard guard(key.device());
  TORCH_CHECK(slot_mapping.scalar_type() == at::kLong && slot_mapping.is_contiguous(),
              "trianglemix: slot_mapping must be contiguous int64");
  const int64_t n = std::min<int64_t>(slot_mapping.numel(), key.size(0));
  check(tmx_reshape_and_cache_fp8(key.data_ptr(), value.data_ptr(), key.stride(0), key.stride(1), fp8_ptr(key_cache),
                                  fp8_ptr(value_cache), key_cache.stride(0), key_cache.stride(1), key_cache.stride(2),
                                  slot_mapping.data_ptr<int64_t>(), (int32_t)n, (int32_t)key.size(1),
                                  (int32_t)key.size(2), (int32_t)key_cache.size(1), dtype_code(key), (float)k_scale,
                                  (float)v_scale, stream_of(key)));
}

void gather_dequant_kv_fp8(Tensor& k_rows, Tensor& v_rows, const Tensor& key_cache, const Tensor& value_cache,
                           const Tensor& block_table, const Tensor& seq_lens, const Tensor& cu_seqlens_k,
                           int64_t max_seq_len, double k_scale, double v_scale) {
  const DeviceGuard guard(key_cache.device());
  TORCH_CHECK(k_rows.is_contiguous() && v_rows.is_contiguous() && k_rows.dim() == 3,
              "trianglemix: k_rows / v_rows must be contiguous [rows, Hkv, D]");
  check(tmx_gather_dequant_kv_fp8(fp8_ptr(key_cache), fp8_ptr(value_cache), key_cache.stride(0), key_cache.stride(1),
                                  key_cache.stride(2), i32(block_table), block_table.stride(0),
                                  (int32_t)key_cache.size(1), i32(seq_lens), i32(cu_seqlens_k),
                                  (int32_t)seq_lens.numel(), (int32_t)max_seq_len, (int32_t)key_cache.size(2),
                                  (int32_t)key_cache.size(3), k_rows.data_ptr(), v_rows.data_ptr(), dtype_code(k_rows),
                                  (float)k_scale, (float)v_scale, stream_of(key_cache)));
}

// ---- 4-bit (MXFP4) cache ----
void on_device(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK(t.device() == like.device(), "trianglemix: ", name, " is on ", t.device(), ", the other tensors on ", like.device());
}

// A pair of 4-bit caches [num_blocks, page_size, Hkv, D / 2 + D / 32]; the head size.
int64_t fp4_caches(const Tensor& k, const Tensor& v) {
  TORCH_CHECK(k.is_cuda(), "trianglemix: the caches must be on a HIP device");
  TORCH_CHECK(k.scalar_type() == at::kByte && v.scalar_type() == at::kByte, "trianglemix: a 4-bit cache is uint8");
  TORCH_CHECK(k.dim() == 4 && k.sizes() == v.sizes() && k.strides() == v.strides(),
              "trianglemix: 4-bit caches must be [num_blocks, page_size, Hkv, D / 2 + D / 32] with equal strides");
  const int64_t width = k.size(3);
  TORCH_CHECK(width == 34 || width == 68, "trianglemix: a 4-bit cache's last dimension is D / 2 + D / 32 with D 64 or 128, not ", width);
  on_device(v, k, "value_cache");
  TORCH_CHECK(k.stride(3) == 1 && k.stride(2) == width && k.stride(1) == k.size(2) * width,
              "trianglemix: a 4-bit page must be one run of bytes (only the page stride is free)");
  return width == 34 ? 64 : 128;
}
void table_rows(const Tensor& block_table, int64_t rows) {
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.stride(1) == 1 && block_table.size(0) >= rows,
              "trianglemix: block_table must be int32 [B, max_blocks] with contiguous rows");
}
void lengths(const Tensor& t, int64_t n, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() && t.numel() >= n, "trianglemix: ", name,
              " must be contiguous int32 with an entry per request");
}

void reshape_and_cache_fp4(const Tensor& key, const Tensor& value, Tensor& key_cache, Tensor& value_cache, const Tensor& slot_mapping) {
  const int64_t d = fp4_caches(key_cache, value_cache);
  const DeviceGuard guard(key_cache.device());
  on_device(key, key_cache, "key");
  on_device(value, key_cache, "value");
  on_device(slot_mapping, key_cache, "slot_mapping");
  TORCH_CHECK(slot_mapping.scalar_type() == at::kLong && slot_mapping.dim() == 1 && slot_mapping.is_contiguous(),
              "trianglemix: slot_mapping must be contiguous int64");
  TORCH_CHECK(key.dim() == 3 && key.sizes() == value.sizes() && key.scalar_type() == value.scalar_type() &&
                  key.size(1) == key_cache.size(2) && key.size(2) == d,
              "trianglemix: key and value must be [T, Hkv, D] rows of one dtype that fit the cache");
  const int64_t n = std::min<int64_t>(slot_mapping.numel(), key.size(0));
  TORCH_CHECK(n == 0 || (key.stride(2) == 1 && value.stride(2) == 1), "trianglemix: the head dimension must be contiguous");
  TORCH_CHECK(n <= 0x7fffffff, "trianglemix: too many rows");
  check(tmx_reshape_and_cache_fp4(key.data_ptr(), value.data_ptr(), key.stride(0), key.stride(1), value.stride(0), value.stride(1),
                                  key_cache.data_ptr(), value_cache.data_ptr(), key_cache.stride(0), key_cache.size(0),
                                  slot_mapping.data_ptr<int64_t>(), (int32_t)n, (int32_t)key.size(1), (int32_t)d,
                                  (int32_t)key_cache.size(1), dtype_code(key), stream_of(key_cache)));
}

void gather_dequant_kv_fp4(Tensor& k_rows, Tensor& v_rows, const Tensor& key_cache, const Tensor& value_cache,
                           const Tensor& block_table, const Tensor& seq_lens, const Tensor& cu_seqlens_k, int64_t total_rows,
                           int64_t max_seq_len) {
  const int64_t d = fp4_caches(key_cache, value_cache);
  const DeviceGuard guard(key_cache.device());
  for (const Tensor* t : {&k_rows, &v_rows}) {
    on_device(*t, key_cache, "out");
    TORCH_CHECK(t->dim() == 3 && t->size(0) >= total_rows && t->size(1) == key_cache.size(2) && t->size(2) == d && t->is_contiguous() &&
                    t->scalar_type() == k_rows.scalar_type(),
                "trianglemix: output rows must be contiguous [>= total_rows, Hkv, D] of one dtype");
  }
  on_device(block_table, key_cache, "block_table");
  on_device(seq_lens, key_cache, "seq_lens");
  on_device(cu_seqlens_k, key_cache, "cu_seqlens_k");
  const int64_t batch = seq_lens.numel();
  lengths(seq_lens, batch, "seq_lens");
  lengths(cu_seqlens_k, batch, "cu_seqlens_k");
  table_rows(block_table, batch);
  TORCH_CHECK(max_seq_len <= 0x7fffffff && block_table.size(1) <= 0x7fffffff && batch <= 0x7fffffff, "trianglemix: sizes past 2^31");
  check(tmx_gather_dequant_kv_fp4(key_cache.data_ptr(), value_cache.data_ptr(), key_cache.stride(0), key_cache.size(0),
                                  block_table.data_ptr<int32_t>(), block_table.stride(0), (int32_t)block_table.size(1),
                                  (int32_t)key_cache.size(1), seq_lens.data_ptr<int32_t>(), cu_seqlens_k.data_ptr<int32_t>(),
                                  (int32_t)batch, (int32_t)max_seq_len, (int32_t)key_cache.size(2), (int32_t)d, k_rows.data_ptr(),
                                  v_rows.data_ptr(), total_rows, dtype_code(k_rows), stream_of(key_cache)));
}

void decode_attention_fp4(Tensor& out, const Tensor& query, const Tensor& key_cache, const Tensor& value_cache, const Tensor& block_table,
                          const Tensor& seq_lens, Tensor& partial_o, Tensor& partial_ml, double scale, int64_t rows_per_request) {
  const int64_t d = fp4_caches(key_cache, value_cache);
  const DeviceGuard guard(key_cache.device());
  on_device(query, key_cache, "q");
  on_device(out, key_cache, "out");
  on_device(block_table, key_cache, "block_table");
  on_device(seq_lens, key_cache, "seq_lens");
  on_device(partial_o, key_cache, "workspace");
  on_device(partial_ml, key_cache, "workspace");
  TORCH_CHECK(query.dim() == 3 && out.sizes() == query.sizes() && query.size(2) == d,
              "trianglemix: q and out must both be [B * rows_per_request, H, D] with the head size of the cache");
  TORCH_CHECK(query.numel() == 0 || (query.stride(2) == 1 && out.stride(2) == 1), "trianglemix: the head dimension must be contiguous");
  TORCH_CHECK(out.scalar_type() == query.scalar_type() || out.scalar_type() == at::kFloat,
              "trianglemix: out must have the dtype of q or be float32");
  const int64_t m = rows_per_request;
  TORCH_CHECK(m >= 1 && m <= 0x7fffffff && query.size(0) % m == 0, "trianglemix: q must hold rows_per_request rows for every request");
  const int64_t batch = query.size(0) / m;
  lengths(seq_lens, batch, "seq_lens");
  table_rows(block_table, batch);
  TORCH_CHECK(partial_o.scalar_type() == at::kFloat && partial_ml.scalar_type() == at::kFloat && partial_o.is_contiguous() &&
                  partial_ml.is_contiguous(),
              "trianglemix: the work area must be contiguous float32 (ops.decode_fp4_workspace)");
  TORCH_CHECK(block_table.size(1) <= 0x7fffffff && batch <= 0x7fffffff, "trianglemix: sizes past 2^31");
  tmx_decode_fp4_args_t a{};
  a.struct_size = sizeof(a);
  a.io_dtype = dtype_code(query);
  a.out_dtype = dtype_code(out);
  a.scale = (float)scale;
  a.batch = (int32_t)batch;
  a.rows_per_request = (int32_t)m;
  a.num_heads = (int32_t)query.size(1);
  a.num_kv_heads = (int32_t)key_cache.size(2);
  a.head_dim = (int32_t)d;
  a.page_size = (int32_t)key_cache.size(1);
  a.out = out.data_ptr();
  a.out_stride_t = out.stride(0);
  a.out_stride_h = out.stride(1);
  a.q = query.data_ptr();
  a.q_stride_t = query.stride(0);
  a.q_stride_h = query.stride(1);
  a.k = key_cache.data_ptr();
  a.v = value_cache.data_ptr();
  a.kv_stride_page = key_cache.stride(0);
  a.num_pages = key_cache.size(0);
  a.block_table = block_table.data_ptr<int32_t>();
  a.block_table_stride = block_table.stride(0);
  a.max_blocks = (int32_t)block_table.size(1);
  a.seq_lens = seq_lens.data_ptr<int32_t>();
  a.partial_o = partial_o.data_ptr<float>();
  a.partial_ml = partial_ml.data_ptr<float>();
  a.workspace_rows = std::min<int64_t>(partial_o.numel() / d, partial_ml.numel() / 2);
  check(tmx_decode_attention_fp4(&a, stream_of(key_cache)));
}

// ---- pages ----
struct PageList {
  std::vector<void*> at;
  int64_t bytes = 16, stride = 16, pages = 0;
};
using TensorRefs = std::vector<const Tensor*>;
TensorRefs refs(const std::vector<Tensor>& v) {
  TensorRefs r;
  r.reserve(v.size());
  for (const Tensor& t : v) r.push_back(&t);
  return r;
}
PageList page_list(const TensorRefs& caches, const Tensor& like) {
  PageList r;
  TORCH_CHECK(like.is_cuda(), "trianglemix: page operators run on HIP devices only");
  if (caches.empty()) return r;
  const Tensor& f = *caches[0];
  TORCH_CHECK(f.dim() >= 2, "trianglemix: a cache is [num_pages, ...]");
  r.at.reserve(caches.size());
  for (const Tensor* t : caches) {
    TORCH_CHECK(t->device() == like.device(), "trianglemix: a cache is on ", t->device(), ", the other tensors on ", like.device());
    TORCH_CHECK(t->scalar_type() == f.scalar_type() && t->sizes() == f.sizes() && t->strides() == f.strides(),
                "trianglemix: the caches must be [num_pages, ...] tensors of one shape, dtype and strides");
    r.at.push_back(t->data_ptr());
  }
  int64_t run = 1;
  for (int64_t i = f.dim() - 1; i >= 1; --i) {
    TORCH_CHECK(f.size(i) == 1 || f.stride(i) == run, "trianglemix: a page must be one run of memory");
    run *= f.size(i);
  }
  r.bytes = run * f.element_size();
  r.pages = f.size(0);
  r.stride = f.size(0) > 1 ? f.stride(0) * f.element_size() : r.bytes;
  return r;
}

void copy_pages(const TensorRefs& caches, const Tensor& pairs) {
  const PageList l = page_list(caches, pairs);
  const DeviceGuard guard(pairs.device());
  TORCH_CHECK((pairs.scalar_type() == at::kInt || pairs.scalar_type() == at::kLong) && pairs.dim() == 2 && pairs.size(1) == 2 &&
                  pairs.is_contiguous() && pairs.size(0) <= 0x7fffffff,
              "trianglemix: pairs must be contiguous int32 or int64 [n, 2]");
  check(tmx_copy_pages(l.at.data(), (int32_t)l.at.size(), l.bytes, l.stride, l.pages, pairs.data_ptr(),
                       pairs.scalar_type() == at::kInt ? 32 : 64, (int32_t)pairs.size(0), nullptr, stream_of(pairs)));
}

void page_table(const Tensor& block_table, const Tensor& seq_lens) {
  TORCH_CHECK(block_table.is_cuda(), "trianglemix: page operators run on HIP devices only");
  table_rows(block_table, seq_lens.numel());
  lengths(seq_lens, seq_lens.numel(), "seq_lens");
  on_device(seq_lens, block_table, "seq_lens");
  TORCH_CHECK(block_table.numel() <= 0x7fffffff, "trianglemix: the block table has more than 2^31 - 1 entries");
}

std::tuple<Tensor, Tensor> free_pages(const Tensor& block_table, const Tensor& seq_lens, int64_t num_pages, int64_t page_size) {
  page_table(block_table, seq_lens);
  const DeviceGuard guard(block_table.device());
  TORCH_CHECK(num_pages >= 0 && num_pages <= (1 << 30) && page_size > 0 && page_size <= (1 << 30), "trianglemix: bad num_pages / page_size");
  const int32_t rows = (int32_t)seq_lens.numel(), cols = (int32_t)block_table.size(1);
  const int64_t work = tmx_pages_work_ints(rows, cols, num_pages);
  Tensor buf = at::empty({num_pages + 1 + work}, block_table.options());
  int32_t* b = buf.data_ptr<int32_t>();
  check(tmx_free_pages(block_table.data_ptr<int32_t>(), block_table.stride(0), rows, cols, seq_lens.data_ptr<int32_t>(), (int32_t)page_size,
                       num_pages, b, b + num_pages, b + num_pages + 1, work, stream_of(block_table)));
  return {buf.narrow(0, 0, num_pages), buf.narrow(0, num_pages, 1)};
}

Tensor fork_pages(const TensorRefs& caches, const Tensor& block_table, const Tensor& seq_lens, const Tensor& parents,
                  const Tensor& fresh, int64_t page_size) {
  page_table(block_table, seq_lens);
  const PageList l = page_list(caches, block_table);
  const DeviceGuard guard(block_table.device());
  lengths(parents, parents.numel(), "parents");
  lengths(fresh, parents.numel(), "fresh");
  on_device(parents, block_table, "parents");
  on_device(fresh, block_table, "fresh");
  TORCH_CHECK(page_size > 0 && page_size <= (1 << 30) && parents.numel() <= 0x7fffffff, "trianglemix: bad page_size or number of children");
  Tensor child = at::empty({parents.numel(), block_table.size(1)}, block_table.options());
  check(tmx_fork_pages(l.at.data(), (int32_t)l.at.size(), l.bytes, l.stride, l.pages, block_table.data_ptr<int32_t>(), block_table.stride(0),
                       (int32_t)seq_lens.numel(), (int32_t)block_table.size(1), seq_lens.data_ptr<int32_t>(), (int32_t)page_size,
                       parents.data_ptr<int32_t>(), fresh.data_ptr<int32_t>(), (int32_t)parents.numel(), child.data_ptr<int32_t>(),
                       stream_of(block_table)));
  return child;
}

std::tuple<Tensor, Tensor> compact_pages(const TensorRefs& caches, const Tensor& block_table, const Tensor& seq_lens,
                                         int64_t page_size) {
  page_table(block_table, seq_lens);
  TORCH_CHECK(!caches.empty(), "trianglemix: compact_pages needs the caches (their first dimension is the pool)");
  const PageList l = page_list(caches, block_table);
  const DeviceGuard guard(block_table.device());
  TORCH_CHECK(page_size > 0 && page_size <= (1 << 30) && l.pages <= (1 << 30), "trianglemix: bad page_size or number of pages");
  const int32_t rows = (int32_t)seq_lens.numel(), cols = (int32_t)block_table.size(1);
  const int64_t work = tmx_pages_work_ints(rows, cols, l.pages), moves = l.pages / 2 + 1;
  // (one allocation for the moves, the totals, the work area and the table that is returned: a second one costs 1.3 us)
  const int64_t table_at = (2 * moves + 2 + work + 63) / 64 * 64;
  Tensor buf = at::empty({table_at + (int64_t)rows * cols}, block_table.options());
  Tensor table = buf.as_strided({rows, cols}, {cols, 1}, table_at);
  int32_t* b = buf.data_ptr<int32_t>();
  check(tmx_plan_compaction(block_table.data_ptr<int32_t>(), block_table.stride(0), rows, cols, seq_lens.data_ptr<int32_t>(),
                            (int32_t)page_size, l.pages, table.data_ptr<int32_t>(), b, b + 2 * moves, b + 2 * moves + 2, work,
                            stream_of(block_table)));
  check(tmx_copy_pages(l.at.data(), (int32_t)l.at.size(), l.bytes, l.stride, l.pages, b, 32, (int32_t)(l.pages / 2), b + 2 * moves + 1,
                       stream_of(block_table)));
  return {table, buf.narrow(0, 2 * moves, 1)};
}

// the registered forms of those that take a list
void copy_pages_op(const std::vector<Tensor>& caches, const Tensor& pairs) { copy_pages(refs(caches), pairs); }
Tensor fork_pages_op(const std::vector<Tensor>& caches, const Tensor& block_table, const Tensor& seq_lens, const Tensor& parents,
                     const Tensor& fresh, int64_t page_size) {
  return fork_pages(refs(caches), block_table, seq_lens, parents, fresh, page_size);
}
std::tuple<Tensor, Tensor> compact_pages_op(const std::vector<Tensor>& caches, const Tensor& block_table, const Tensor& seq_lens,
                                            int64_t page_size) {
  return compact_pages(refs(caches), block_table, seq_lens, page_size);
}

}  // namespace

TORCH_LIBRARY(_trianglemix_C, m) {
  m.def("trianglemix_index_sizes(Tensor cu_seqlens_q_cpu, Tensor seq_lens_cpu, int si, int sl, int last, int block_m, "
        "int block_n, int mode, int tri_min_len, int chunk_tiles, Tensor? full_lens_cpu=None, int dense_rows_from=0) -> int[]");
  m.impl("trianglemix_index_sizes", c10::DispatchKey::CPU, &index_sizes);
  m.def("trianglemix_suggest_chunk_tiles(Tensor cu_seqlens_q_cpu, Tensor seq_lens_cpu, int si, int sl, int last, "
        "int block_m, int block_n, int mode, int tri_min_len, int units_per_item, int num_cus, "
        "Tensor? full_lens_cpu=None) -> int");
  m.impl("trianglemix_suggest_chunk_tiles", c10::DispatchKey::CPU, &suggest_chunk_tiles);
  m.def("trianglemix_build_block_index(Tensor(a!)[] index, Tensor? tile_pages, Tensor cu_seqlens_q, Tensor seq_lens, "
        "Tensor cu_seqlens_q_cpu, Tensor seq_lens_cpu, Tensor? block_table, int page_size, int si, int sl, int last, "
        "int block_m, int block_n, int mode, int tri_min_len, int chunk_tiles, Tensor? full_lens=None, "
        "Tensor? full_lens_cpu=None, int dense_rows_from=0) -> ()");
  m.impl("trianglemix_build_block_index", c10::DispatchKey::CUDA, &build_block_index);
  m.def("trianglemix_attention(Tensor! out, Tensor query, Tensor key_cache, Tensor value_cache, Tensor? block_table, "
        "Tensor cu_seqlens_q, Tensor seq_lens, Tensor? cu_seqlens_k, Tensor[] index, Tensor? tile_pages, "
        "Tensor? partial_o, Tensor? partial_ml, Tensor? bias, float scale, int si, int sl, int last, int mode, "
        "int tri_min_len, int chunk_tiles, int num_items, int num_partials, int num_split_qblocks, "
        "Tensor? full_lens=None, int flags=0, int nnz_tiles=0, Tensor? k_new=None, Tensor? v_new=None, "
        "Tensor? cache_slots=None, float k_scale=1.0, float v_scale=1.0, int index_block_m=0, int index_block_n=0, "
        "Tensor? kv_stage=None, int index_dense_rows_from=0) -> ()");
  m.impl("trianglemix_attention", c10::DispatchKey::CUDA, &attention);
  m.def("trianglemix_decode_attention(Tensor! out, Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, "
        "Tensor seq_lens, Tensor! partial_o, Tensor! partial_ml, float scale, Tensor? k_new=None, Tensor? v_new=None, "
        "Tensor? cache_slots=None, float k_scale=1.0, float v_scale=1.0) -> ()");
  m.impl("trianglemix_decode_attention", c10::DispatchKey::CUDA, &decode_attention);
  m.def("trianglemix_reshape_and_cache(Tensor key, Tensor value, Tensor! key_cache, Tensor! value_cache, "
        "Tensor slot_mapping) -> ()");
  m.impl("trianglemix_reshape_and_cache", c10::DispatchKey::CUDA, &reshape_and_cache);
  m.def("trianglemix_reshape_and_cache_fp8(Tensor key, Tensor value, Tensor! key_cache, Tensor! value_cache, "
        "Tensor slot_mapping, float k_scale, float v_scale) -> ()");
  m.impl("trianglemix_reshape_and_cache_fp8", c10::DispatchKey::CUDA, &reshape_and_cache_fp8);
  m.def("trianglemix_gather_dequant_kv_fp8(Tensor! k_rows, Tensor! v_rows, Tensor key_cache, Tensor value_cache, "
        "Tensor block_table, Tensor seq_lens, Tensor cu_seqlens_k, int max_seq_len, float k_scale, float v_scale) -> ()");
  m.impl("trianglemix_gather_dequant_kv_fp8", c10::DispatchKey::CUDA, &gather_dequant_kv_fp8);
  m.def("trianglemix_reshape_and_cache_fp4(Tensor key, Tensor value, Tensor! key_cache, Tensor! value_cache, "
        "Tensor slot_mapping) -> ()");
  m.impl("trianglemix_reshape_and_cache_fp4", c10::DispatchKey::CUDA, &reshape_and_cache_fp4);
  m.def("trianglemix_gather_dequant_kv_fp4(Tensor! k_rows, Tensor! v_rows, Tensor key_cache, Tensor value_cache, "
        "Tensor block_table, Tensor seq_lens, Tensor cu_seqlens_k, int total_rows, int max_seq_len) -> ()");
  m.impl("trianglemix_gather_dequant_kv_fp4", c10::DispatchKey::CUDA, &gather_dequant_kv_fp4);
  m.def("trianglemix_decode_attention_fp4(Tensor! out, Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, "
        "Tensor seq_lens, Tensor! partial_o, Tensor! partial_ml, float scale, int rows_per_request=1) -> ()");
  m.impl("trianglemix_decode_attention_fp4", c10::DispatchKey::CUDA, &decode_attention_fp4);
  m.def("trianglemix_copy_pages(Tensor(a!)[] caches, Tensor pairs) -> ()");
  m.impl("trianglemix_copy_pages", c10::DispatchKey::CUDA, &copy_pages_op);
  m.def("trianglemix_free_pages(Tensor block_table, Tensor seq_lens, int num_pages, int page_size) -> (Tensor, Tensor)");
  m.impl("trianglemix_free_pages", c10::DispatchKey::CUDA, &free_pages);
  m.def("trianglemix_fork_pages(Tensor(a!)[] caches, Tensor block_table, Tensor seq_lens, Tensor parents, Tensor fresh, "
        "int page_size) -> Tensor");
  m.impl("trianglemix_fork_pages", c10::DispatchKey::CUDA, &fork_pages_op);
  m.def("trianglemix_compact_pages(Tensor(a!)[] caches, Tensor block_table, Tensor seq_lens, int page_size) -> (Tensor, Tensor)");
  m.impl("trianglemix_compact_pages", c10::DispatchKey::CUDA, &compact_pages_op);
}

// The extension is also a Python module, so that a plain `import` of the shared object runs the
// TORCH_LIBRARY block above: the reference's REGISTER_EXTENSION (csrc/core/registration.h:13-27), which is
// how vllm/platforms/rocm.py:32-40 loads vllm._C / vllm._rocm_C.
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/record_function.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

// The page operators are also plain functions of the module (same names without the prefix, positional arguments): turning
// a Python list of 72 tensors into the registry's own costs 5.2 us of a call's 10.7, reading it in place 0.2 us, and outputs
// made below the autograd keys, as in the registry's kernels, are handed to Python as they are (free_pages 6.2 -> 4.8 us).
// (Calls that only fill their arguments gain nothing: they stay with the registry.)  They serve plain tensors that nothing
// watches.  With a dispatch or function mode, a tensor subclass (a fake tensor has no memory to work on), a functorch
// transform or a profiler about, they do nothing and return NotImplemented: the caller then goes through the registry, which
// these see.
namespace {

const c10::DispatchKeySet kWatchers(
    {c10::DispatchKey::Python, c10::DispatchKey::PythonDispatcher, c10::DispatchKey::Functionalize, c10::DispatchKey::Tracer,
     c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchVmapMode, c10::DispatchKey::FuncTorchGradWrapper,
     c10::DispatchKey::FuncTorchDynamicLayerFrontMode, c10::DispatchKey::FuncTorchDynamicLayerBackMode});

struct Args {
  PyObject* const* at;
  Py_ssize_t n, next = 0;
  bool watched = at::hasCallbacks() || at::impl::torch_function_mode_enabled() ||
                 c10::impl::tls_local_dispatch_key_set().included_.has_any(kWatchers);
  Args(PyObject* const* at, Py_ssize_t n, Py_ssize_t takes) : at(at), n(n) {
    TORCH_CHECK(n == takes, "trianglemix: the operator takes ", takes, " arguments, not ", n);
  }
  PyObject* take() { return at[next++]; }
  const Tensor& variable(PyObject* o) {
    const Tensor& t = THPVariable_Unpack(o);
    watched = watched || t.key_set().has_any(kWatchers) || !THPVariable_CheckExact(o);
    return t;
  }
  const Tensor& tensor() {
    PyObject* o = take();
    TORCH_CHECK(THPVariable_Check(o), "trianglemix: argument ", next, " must be a tensor");
    return variable(o);
  }
  int64_t integer() {
    PyObject* o = take();
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
  }
  TensorRefs tensors() {
    PyObject* o = take();
    TORCH_CHECK(PyList_Check(o) || PyTuple_Check(o), "trianglemix: argument ", next, " must be a list or tuple of tensors");
    const Py_ssize_t k = PySequence_Fast_GET_SIZE(o);
    PyObject** items = PySequence_Fast_ITEMS(o);
    TensorRefs r;
    r.reserve((size_t)k);
    for (Py_ssize_t i = 0; i < k; ++i) {
      TORCH_CHECK(THPVariable_Check(items[i]), "trianglemix: argument ", next, " must hold tensors only");
      r.push_back(&variable(items[i]));
    }
    return r;
  }
};

PyObject* two(const std::tuple<Tensor, Tensor>& t) {
  PyObject* a = THPVariable_Wrap(std::get<0>(t));
  PyObject* b = THPVariable_Wrap(std::get<1>(t));
  PyObject* r = a && b ? PyTuple_Pack(2, a, b) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  return r;
}

PyObject* py_copy_pages(PyObject*, PyObject* const* at, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{at, n, 2};
  const TensorRefs caches = a.tensors();
  const Tensor& pairs = a.tensor();
  if (a.watched) Py_RETURN_NOTIMPLEMENTED;
  copy_pages(caches, pairs);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
PyObject* py_fork_pages(PyObject*, PyObject* const* at, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{at, n, 6};
  const TensorRefs caches = a.tensors();
  const Tensor &bt = a.tensor(), &sl = a.tensor(), &parents = a.tensor(), &fresh = a.tensor();
  const int64_t page_size = a.integer();
  if (a.watched) Py_RETURN_NOTIMPLEMENTED;
  const at::AutoDispatchBelowADInplaceOrView below;
  return THPVariable_Wrap(fork_pages(caches, bt, sl, parents, fresh, page_size));
  END_HANDLE_TH_ERRORS
}
PyObject* py_free_pages(PyObject*, PyObject* const* at, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{at, n, 4};
  const Tensor &bt = a.tensor(), &sl = a.tensor();
  const int64_t pages = a.integer(), page_size = a.integer();
  if (a.watched) Py_RETURN_NOTIMPLEMENTED;
  const at::AutoDispatchBelowADInplaceOrView below;
  return two(free_pages(bt, sl, pages, page_size));
  END_HANDLE_TH_ERRORS
}
PyObject* py_compact_pages(PyObject*, PyObject* const* at, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a{at, n, 4};
  const TensorRefs caches = a.tensors();
  const Tensor &bt = a.tensor(), &sl = a.tensor();
  const int64_t page_size = a.integer();
  if (a.watched) Py_RETURN_NOTIMPLEMENTED;
  const at::AutoDispatchBelowADInplaceOrView below;
  return two(compact_pages(caches, bt, sl, page_size));
  END_HANDLE_TH_ERRORS
}

#define TMX_PY(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&py_##name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {TMX_PY(copy_pages), TMX_PY(fork_pages), TMX_PY(compact_pages), TMX_PY(free_pages), {nullptr, nullptr, 0, nullptr}};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__trianglemix_C() {
  static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_trianglemix_C", nullptr, 0, methods};
  return PyModule_Create(&module);
}
