// C ABI of the 8-bit paged cache (include/b200_paged.h, section 7): argument checks and launches.
#include "api_common.cuh"
#include "fp8.cuh"
#include "fp8_decode.cuh"
#include "nvtx.cuh"

using b200::cuda_fail;
using b200::esize_of;
using b200::fail;
using b200::num_sms;

namespace {

int check_cache(const B200Fp8Cache* c, int dtype) {
  if (c == nullptr) return fail(B200_ERR_INVALID_ARGUMENT, "null cache");
  if (esize_of(dtype) == 0) return fail(B200_ERR_UNSUPPORTED, "unsupported dtype");
  if (c->num_layers <= 0 || c->total_blocks <= 0 || c->block_size <= 0 || c->num_kv_heads <= 0 ||
      c->head_dim <= 0)
    return fail(B200_ERR_INVALID_ARGUMENT, "cache geometry must be positive");
  if (c->layer_idx < 0 || c->layer_idx >= c->num_layers)
    return fail(B200_ERR_INVALID_ARGUMENT, "layer_idx out of range");
  if (c->block_size > 1024) return fail(B200_ERR_UNSUPPORTED, "block_size > 1024");
  if (c->head_dim > 256) return fail(B200_ERR_UNSUPPORTED, "head_dim > 256");
  if (c->num_kv_heads > 1024) return fail(B200_ERR_UNSUPPORTED, "num_kv_heads > 1024");
  return B200_OK;
}

bool has_arrays(const B200Fp8Cache& c) {
  return c.key_cache && c.value_cache && c.key_scale && c.value_scale;
}

// Cache side of an append, and its scratch in the caller's workspace.
int append_args(const B200Fp8Cache& c, const int64_t* slots, int32_t n, void* workspace,
                size_t workspace_bytes, int32_t* status, b200::AppendFp8Args* a) {
  a->kc = static_cast<uint8_t*>(c.key_cache);
  a->vc = static_cast<uint8_t*>(c.value_cache);
  a->ks = c.key_scale;
  a->vs = c.value_scale;
  a->layer = c.layer_idx;
  a->nb = c.total_blocks;
  a->bs = c.block_size;
  a->hkv = c.num_kv_heads;
  a->head_dim = c.head_dim;
  a->slots = slots;
  a->num_tokens = n;
  a->status = status;
  const size_t need = b200::append_fp8_scratch_bytes(c.total_blocks, n);
  if (need == 0) return B200_OK;
  if (workspace == nullptr || workspace_bytes < need)
    return fail(B200_ERR_INVALID_ARGUMENT, "append workspace too small");
  if (reinterpret_cast<uintptr_t>(workspace) % 4 != 0)
    return fail(B200_ERR_INVALID_ARGUMENT, "append workspace must be 4-byte aligned");
  a->count = static_cast<int32_t*>(workspace);
  a->first = a->count + c.total_blocks;
  a->num_runs = a->first + c.total_blocks;
  a->runs = a->num_runs + 1;
  return B200_OK;
}

int check_attention(const B200AttentionFp8Params* p) {
  if (p == nullptr) return fail(B200_ERR_INVALID_ARGUMENT, "null params");
  const int rc = check_cache(&p->cache, p->dtype);
  if (rc != B200_OK) return rc;
  if (p->num_query_heads <= 0 || p->num_query_heads % p->cache.num_kv_heads != 0)
    return fail(B200_ERR_INVALID_ARGUMENT,
                "num_query_heads must be a multiple of num_kv_heads for GQA");
  if (p->num_seqs < 0 || p->num_tokens < 0)
    return fail(B200_ERR_INVALID_ARGUMENT, "negative sizes");
  if (p->block_table_stride < 0)
    return fail(B200_ERR_INVALID_ARGUMENT, "negative block_table_stride");
  return B200_OK;
}

b200::AttnFp8Args attention_args(const B200AttentionFp8Params& p) {
  b200::AttnFp8Args a{};
  const B200Fp8Cache& c = p.cache;
  a.q = p.query;
  a.q_srow = p.q_stride_row;
  a.q_shead = p.q_stride_head;
  a.kc = static_cast<const uint8_t*>(c.key_cache);
  a.vc = static_cast<const uint8_t*>(c.value_cache);
  a.ks = c.key_scale;
  a.vs = c.value_scale;
  a.layer = c.layer_idx;
  a.nb = c.total_blocks;
  a.bs = c.block_size;
  a.hkv = c.num_kv_heads;
  a.head_dim = c.head_dim;
  a.hq = p.num_query_heads;
  a.group = p.num_query_heads / c.num_kv_heads;
  a.bt = p.block_tables;
  a.bt_stride = p.block_table_stride;
  a.ctx_lens = p.context_lens;
  a.S = p.num_seqs;
  a.scale = p.scale;
  a.out = p.out;
  a.o_srow = p.o_stride_row;
  a.o_shead = p.o_stride_head;
  a.status = p.status_word;
  return a;
}

size_t align256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

// One launch of the tensor-core decode (up to kDecodeFp8MaxSeqs sequences) and its workspace.
struct DecodePlan {
  bool tensor_cores;
  int nchunks, grid;
  int64_t max_ctx;
  size_t off_ml, off_o, total;
};

DecodePlan decode_plan(const B200AttentionFp8Params& p) {
  const B200Fp8Cache& c = p.cache;
  DecodePlan pl{};
  const int64_t rows = static_cast<int64_t>(c.num_layers) * c.total_blocks * c.block_size;
  pl.tensor_cores = (c.head_dim == 64 || c.head_dim == 128) &&
                    (c.block_size == 8 || c.block_size % 16 == 0) && rows < (int64_t(1) << 31) &&
                    reinterpret_cast<uintptr_t>(c.key_cache) % 16 == 0 &&
                    reinterpret_cast<uintptr_t>(c.value_cache) % 16 == 0;
  if (!pl.tensor_cores) return pl;
  const int group = p.num_query_heads / c.num_kv_heads;
  pl.nchunks = (group + 7) / 8;
  const int S = p.num_seqs < b200::kDecodeFp8MaxSeqs ? p.num_seqs : b200::kDecodeFp8MaxSeqs;
  // no sequence reaches past its row of the table
  pl.max_ctx = p.max_context_len;
  const int64_t most = static_cast<int64_t>(p.block_table_stride) * c.block_size;
  if (pl.max_ctx > most) pl.max_ctx = most;
  if (pl.max_ctx < 0) pl.max_ctx = 0;
  pl.grid = b200::decode_fp8_grid(S, pl.max_ctx, c.num_kv_heads * pl.nchunks, num_sms());
  const size_t parts = b200::decode_fp8_parts(pl.grid);
  pl.off_ml = align256(parts / 2 * sizeof(b200::MergeItem));
  pl.off_o = pl.off_ml + align256(parts * 8 * sizeof(float2));
  pl.total = pl.off_o + align256(parts * 8 * c.head_dim * sizeof(float));
  return pl;
}

// A cache (L, NB, BS, Hkv, D) of bytes as (D, Hkv, L*NB*BS), box (D, 1, box_rows), swizzled over
// the D bytes of a row.
int code_map(const void* cache, const B200Fp8Cache& c, int box_rows, CUtensorMap* out) {
  b200::EncodeTiledFn fn = b200::encode_fn();
  if (fn == nullptr) return fail(B200_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const cuuint64_t D = c.head_dim, H = c.num_kv_heads;
  const cuuint64_t dims[3] = {D, H, static_cast<cuuint64_t>(c.num_layers) * c.total_blocks * c.block_size};
  const cuuint64_t strides[2] = {D, H * D};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(D), 1, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r =
      fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(cache), dims, strides, box, estr,
         CU_TENSOR_MAP_INTERLEAVE_NONE,
         c.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(B200_ERR_CUDA, "cuTensorMapEncodeTiled failed");
  return B200_OK;
}

// cu_q: mixed batch, only sequences with exactly one new token are decoded (row cu_q[s]).
int run_decode(const B200AttentionFp8Params& p, const DecodePlan& pl, const int64_t* cu_q,
               bool decodes_only, char* ws, cudaStream_t st) {
  const B200Fp8Cache& c = p.cache;
  CUtensorMap km, vm;
  const int box_rows = c.block_size >= 16 ? 16 : 8;
  int rc = code_map(c.key_cache, c, box_rows, &km);
  if (rc == B200_OK) rc = code_map(c.value_cache, c, box_rows, &vm);
  if (rc != B200_OK) return rc;
  b200::DecodeFp8Args a{};
  a.q_srow = p.q_stride_row;
  a.q_shead = p.q_stride_head;
  a.ks = c.key_scale;
  a.vs = c.value_scale;
  a.layer = c.layer_idx;
  a.nb = c.total_blocks;
  a.bs = c.block_size;
  a.hkv = c.num_kv_heads;
  a.head_dim = c.head_dim;
  a.group = p.num_query_heads / c.num_kv_heads;
  a.nchunks = pl.nchunks;
  a.bt_stride = p.block_table_stride;
  a.max_ctx = static_cast<int32_t>(pl.max_ctx);
  a.scale_log2 = p.scale * b200::kLog2e;
  a.o_srow = p.o_stride_row;
  a.o_shead = p.o_stride_head;
  a.decodes_only = decodes_only ? 1 : 0;
  a.status = p.status_word;
  a.merge = reinterpret_cast<b200::MergeItem*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + pl.off_ml);
  a.part_o = reinterpret_cast<float*>(ws + pl.off_o);
  for (int s0 = 0; s0 < p.num_seqs; s0 += b200::kDecodeFp8MaxSeqs) {
    a.S = p.num_seqs - s0 < b200::kDecodeFp8MaxSeqs ? p.num_seqs - s0 : b200::kDecodeFp8MaxSeqs;
    a.bt = p.block_tables + static_cast<int64_t>(s0) * p.block_table_stride;
    a.ctx_lens = p.context_lens + s0;
    a.cu_q = cu_q ? cu_q + s0 : nullptr;
    a.query_rows = !cu_q && p.query_rows ? p.query_rows + s0 : nullptr;
    // without a map, sequence s reads and writes row s of the call
    const int64_t shift = cu_q || p.query_rows ? 0 : s0;
    a.q = static_cast<const char*>(p.query) + shift * p.q_stride_row * esize_of(p.dtype);
    const size_t four = 4 * esize_of(p.dtype);
    a.vec_q = reinterpret_cast<uintptr_t>(a.q) % four == 0 && a.q_srow % 4 == 0 && a.q_shead % 4 == 0;
    a.out = static_cast<char*>(p.out) + shift * p.o_stride_row * esize_of(p.dtype);
    const cudaError_t e = b200::launch_decode_fp8(p.dtype, km, vm, a, pl.grid, st);
    if (e != cudaSuccess) return cuda_fail(e, "paged_decode_fp8");
  }
  return B200_OK;
}

int check_workspace(const void* ws, size_t have, size_t need) {
  if (need == 0) return B200_OK;
  if (ws == nullptr || have < need) return fail(B200_ERR_INVALID_ARGUMENT, "attention workspace too small");
  if (reinterpret_cast<uintptr_t>(ws) % 256 != 0)
    return fail(B200_ERR_INVALID_ARGUMENT, "attention workspace must be 256-byte aligned");
  return B200_OK;
}

// A prefill on the tensor cores: the decode's workspace, the 16-bit copy of the pages of the
// sequences with more than one new token, and the 16-bit prefill's own workspace.
struct PrefillPlan {
  bool tensor_cores;
  DecodePlan decode;
  int32_t blocks, stride, max_ctx;
  size_t off_ctx, off_table, off_chunks, chunk_bytes, off_k, off_v, total;
};

// The 16-bit prefill's parameters over the copy at `ws`.
B200PrefillParams chunk_params(const B200AttentionFp8Params& p, const PrefillPlan& pl, char* ws) {
  B200PrefillParams c{};
  c.query = p.query;
  c.q_stride_token = p.q_stride_row;
  c.q_stride_head = p.q_stride_head;
  c.key_cache = ws + pl.off_k;
  c.value_cache = ws + pl.off_v;
  c.geom = {1, pl.blocks, p.cache.block_size, p.cache.num_kv_heads, p.cache.head_dim, p.dtype};
  c.layer_idx = 0;
  c.num_query_heads = p.num_query_heads;
  c.block_tables = reinterpret_cast<int32_t*>(ws + pl.off_table);
  c.block_table_stride = pl.stride;
  c.cu_seqlens = p.cu_seqlens;
  c.context_lens = reinterpret_cast<int32_t*>(ws + pl.off_ctx);
  c.num_seqs = p.num_seqs;
  c.num_tokens = p.num_tokens;
  c.max_query_len = p.max_query_len;
  c.max_context_len = pl.max_ctx;
  c.scale = p.scale;
  c.out = p.out;
  c.o_stride_token = p.o_stride_row;
  c.o_stride_head = p.o_stride_head;
  c.status_word = p.status_word;
  return c;
}

PrefillPlan prefill_plan(const B200AttentionFp8Params& p) {
  PrefillPlan pl{};
  pl.decode = decode_plan(p);
  const B200Fp8Cache& c = p.cache;
  if (!pl.decode.tensor_cores || p.dtype == B200_DTYPE_F32) return pl;
  pl.max_ctx = static_cast<int32_t>(pl.decode.max_ctx);
  pl.stride = (pl.max_ctx + c.block_size - 1) / c.block_size;
  if (pl.stride < 1) pl.stride = 1;
  // at most half of the new tokens begin a sequence with more than one
  const int64_t seqs = p.num_seqs < p.num_tokens / 2 ? p.num_seqs : p.num_tokens / 2;
  int64_t blocks = seqs * pl.stride;
  if (p.prefill_blocks >= 0 && p.prefill_blocks < blocks) blocks = p.prefill_blocks;
  const int64_t block_bytes = static_cast<int64_t>(c.block_size) * c.num_kv_heads * c.head_dim * 2;
  if (blocks > (int64_t(1) << 31) / c.block_size - 1) return pl;  // rows of the copy pass 31 bits
  pl.blocks = blocks < 1 ? 1 : static_cast<int32_t>(blocks);
  pl.chunk_bytes = b200::prefill_chunks_workspace_bytes(chunk_params(p, pl, nullptr));
  if (pl.chunk_bytes == 0) return pl;
  pl.tensor_cores = true;
  size_t off = align256(pl.decode.total);
  const auto take = [&off](size_t bytes) {
    const size_t at = off;
    off += align256(bytes);
    return at;
  };
  pl.off_ctx = take(static_cast<size_t>(p.num_seqs) * 4);
  pl.off_table = take(static_cast<size_t>(p.num_seqs) * pl.stride * 4);
  pl.off_chunks = take(pl.chunk_bytes);
  pl.off_k = take(static_cast<size_t>(pl.blocks) * block_bytes);
  pl.off_v = take(static_cast<size_t>(pl.blocks) * block_bytes);
  pl.total = off;
  return pl;
}

// Decode of the one-token sequences, the copy, and the prefill of the others over it, whose products
// with V take the softmax weights in the query's type as its tensor-core operands have to be
// (bf16: 2.2e-3 off 64 bits in the mean, 1.7e-3 being the outputs' own rounding).  Copying
// costs 3 bytes of traffic per cached entry once, against 4 G D flops per entry and new token.
// A step of 16 chunks of 128 to 2048 tokens on up to 2048 cached ones and 240 decodes (GQA 32/8, D 128):
// decode 130 us, copy 44, plan 9, prefill 458 (0.95 PFLOP/s); a CTA per query row took 121 ms, and one
// prompt of 8192 150 ms against 0.53.
int run_prefill(const B200AttentionFp8Params& p, const PrefillPlan& pl, char* ws, cudaStream_t st) {
  // by the caller's bounds there is nothing but decodes
  const bool decodes_only = p.num_tokens < 2 || p.max_query_len < 2 || p.prefill_blocks == 0;
  const int rc = run_decode(p, pl.decode, p.cu_seqlens, decodes_only, ws, st);
  if (rc != B200_OK || decodes_only) return rc;
  const B200Fp8Cache& c = p.cache;
  b200::ExpandFp8Args a{};
  a.kc = static_cast<const uint8_t*>(c.key_cache);
  a.vc = static_cast<const uint8_t*>(c.value_cache);
  a.ks = c.key_scale;
  a.vs = c.value_scale;
  a.layer = c.layer_idx;
  a.nb = c.total_blocks;
  a.bs = c.block_size;
  a.hkv = c.num_kv_heads;
  a.head_dim = c.head_dim;
  a.bt = p.block_tables;
  a.bt_stride = p.block_table_stride;
  a.ctx_lens = p.context_lens;
  a.cu_q = p.cu_seqlens;
  a.S = p.num_seqs;
  a.max_ctx = pl.max_ctx;
  a.scratch_blocks = pl.blocks;
  a.scratch_stride = pl.stride;
  a.scratch_ctx = reinterpret_cast<int32_t*>(ws + pl.off_ctx);
  a.scratch_table = reinterpret_cast<int32_t*>(ws + pl.off_table);
  a.k16 = ws + pl.off_k;
  a.v16 = ws + pl.off_v;
  a.status = p.status_word;
  const cudaError_t e = b200::launch_expand_fp8(a, p.dtype, num_sms(), st);
  if (e != cudaSuccess) return cuda_fail(e, "prefill_fp8 copy");
  return b200::prefill_chunks(chunk_params(p, pl, ws), ws + pl.off_chunks, pl.chunk_bytes, st);
}

bool has_arrays(const B200AttentionFp8Params& p) {
  return has_arrays(p.cache) && p.query && p.out && p.block_tables && p.context_lens;
}

}  // namespace

extern "C" {

size_t b200_append_fp8_workspace_bytes(const B200Fp8Cache* cache, int32_t num_tokens) {
  if (cache == nullptr || cache->total_blocks <= 0 || num_tokens <= 0) return 0;
  return b200::append_fp8_scratch_bytes(cache->total_blocks, num_tokens);
}

int b200_reshape_and_cache_fp8(const B200Fp8Cache* cache, int32_t dtype, const void* key,
                               int64_t k_stride_token, int64_t k_stride_head, const void* value,
                               int64_t v_stride_token, int64_t v_stride_head,
                               const int64_t* slot_mapping, int32_t num_tokens, void* workspace,
                               size_t workspace_bytes, int32_t* status_word, void* stream) {
  b200::NvtxRange nvtx_range("b200_reshape_and_cache_fp8");
  int rc = check_cache(cache, dtype);
  if (rc != B200_OK) return rc;
  if (num_tokens < 0) return fail(B200_ERR_INVALID_ARGUMENT, "num_tokens < 0");
  if (num_tokens == 0) return B200_OK;
  if (!has_arrays(*cache) || !key || !value || !slot_mapping)
    return fail(B200_ERR_INVALID_ARGUMENT, "null pointer");
  b200::AppendFp8Args a{};
  rc = append_args(*cache, slot_mapping, num_tokens, workspace, workspace_bytes, status_word, &a);
  if (rc != B200_OK) return rc;
  a.key = key;
  a.value = value;
  a.k_stok = k_stride_token;
  a.k_shead = k_stride_head;
  a.v_stok = v_stride_token;
  a.v_shead = v_stride_head;
  cudaError_t e =
      b200::launch_append_fp8(a, dtype, num_sms(), static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "reshape_and_cache_fp8");
  return B200_OK;
}

int b200_rope_reshape_and_cache_fp8(const B200Fp8Cache* cache, int32_t dtype, const void* qkv,
                                    int64_t qkv_stride_token, int32_t num_tokens,
                                    int32_t num_query_heads, const int64_t* positions,
                                    const float* inv_freq, void* q_out,
                                    int64_t q_out_stride_token, const int64_t* slot_mapping,
                                    void* workspace, size_t workspace_bytes,
                                    int32_t* status_word, void* stream) {
  b200::NvtxRange nvtx_range("b200_rope_reshape_and_cache_fp8");
  int rc = check_cache(cache, dtype);
  if (rc != B200_OK) return rc;
  const int D = cache->head_dim, hkv = cache->num_kv_heads;
  if (D % 2 != 0) return fail(B200_ERR_INVALID_ARGUMENT, "head_dim must be even");
  if (num_query_heads <= 0 || num_query_heads % hkv != 0)
    return fail(B200_ERR_INVALID_ARGUMENT, "num_query_heads must be a multiple of num_kv_heads");
  if (num_tokens < 0) return fail(B200_ERR_INVALID_ARGUMENT, "num_tokens < 0");
  if (num_tokens == 0) return B200_OK;
  if (qkv_stride_token < static_cast<int64_t>(num_query_heads + 2 * hkv) * D && num_tokens > 1)
    return fail(B200_ERR_INVALID_ARGUMENT, "qkv_stride_token shorter than a q,k,v row");
  if (q_out_stride_token < static_cast<int64_t>(num_query_heads) * D && num_tokens > 1)
    return fail(B200_ERR_INVALID_ARGUMENT, "q_out_stride_token shorter than a q row");
  if (!has_arrays(*cache) || !qkv || !positions || !inv_freq || !q_out || !slot_mapping)
    return fail(B200_ERR_INVALID_ARGUMENT, "null pointer");
  b200::AppendFp8Args a{};
  rc = append_args(*cache, slot_mapping, num_tokens, workspace, workspace_bytes, status_word, &a);
  if (rc != B200_OK) return rc;
  const int es = esize_of(dtype);
  a.q_in = qkv;
  a.q_stok = qkv_stride_token;
  a.q_out = q_out;
  a.qo_stok = q_out_stride_token;
  a.hq = num_query_heads;
  a.key = static_cast<const char*>(qkv) + static_cast<int64_t>(num_query_heads) * D * es;
  a.value = static_cast<const char*>(a.key) + static_cast<int64_t>(hkv) * D * es;
  a.k_stok = a.v_stok = qkv_stride_token;
  a.k_shead = a.v_shead = D;
  a.positions = positions;
  a.inv_freq = inv_freq;
  cudaError_t e =
      b200::launch_append_fp8(a, dtype, num_sms(), static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "rope_reshape_and_cache_fp8");
  return B200_OK;
}

int b200_gather_cache_fp8(const B200Fp8Cache* cache, int32_t dtype, const int64_t* slots,
                          int64_t n, void* k_out, void* v_out, int32_t* status_word,
                          void* stream) {
  b200::NvtxRange nvtx_range("b200_gather_cache_fp8");
  const int rc = check_cache(cache, dtype);
  if (rc != B200_OK) return rc;
  if (n < 0) return fail(B200_ERR_INVALID_ARGUMENT, "n < 0");
  if (n == 0) return B200_OK;
  if (!has_arrays(*cache) || !slots || !k_out || !v_out)
    return fail(B200_ERR_INVALID_ARGUMENT, "null pointer");
  b200::GatherFp8Args a{};
  a.kc = static_cast<const uint8_t*>(cache->key_cache);
  a.vc = static_cast<const uint8_t*>(cache->value_cache);
  a.ks = cache->key_scale;
  a.vs = cache->value_scale;
  a.layer = cache->layer_idx;
  a.nb = cache->total_blocks;
  a.bs = cache->block_size;
  a.hkv = cache->num_kv_heads;
  a.head_dim = cache->head_dim;
  a.slots = slots;
  a.n = n;
  a.k_out = k_out;
  a.v_out = v_out;
  a.status = status_word;
  cudaError_t e =
      b200::launch_gather_fp8(a, dtype, num_sms(), static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "gather_cache_fp8");
  return B200_OK;
}

size_t b200_paged_decode_fp8_workspace_bytes(const B200AttentionFp8Params* p) {
  if (check_attention(p) != B200_OK || p->num_seqs == 0) return 0;
  return decode_plan(*p).total;
}

int b200_paged_decode_fp8(const B200AttentionFp8Params* p, void* workspace,
                          size_t workspace_bytes, void* stream) {
  b200::NvtxRange nvtx_range("b200_paged_decode_fp8");
  int rc = check_attention(p);
  if (rc != B200_OK) return rc;
  if (p->num_seqs == 0) return B200_OK;
  if (!has_arrays(*p)) return fail(B200_ERR_INVALID_ARGUMENT, "null pointer");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const DecodePlan pl = decode_plan(*p);
  if (pl.tensor_cores) {
    rc = check_workspace(workspace, workspace_bytes, pl.total);
    if (rc != B200_OK) return rc;
    return run_decode(*p, pl, nullptr, false, static_cast<char*>(workspace), st);
  }
  b200::AttnFp8Args a = attention_args(*p);
  a.query_rows = p->query_rows;
  const cudaError_t e = b200::launch_row_fp8(a, p->dtype, p->num_seqs, st);
  if (e != cudaSuccess) return cuda_fail(e, "paged_decode_fp8");
  return B200_OK;
}

size_t b200_paged_prefill_fp8_workspace_bytes(const B200AttentionFp8Params* p) {
  if (check_attention(p) != B200_OK || p->num_seqs == 0 || p->num_tokens == 0) return 0;
  return prefill_plan(*p).total;
}

int b200_paged_prefill_fp8(const B200AttentionFp8Params* p, void* workspace,
                           size_t workspace_bytes, void* stream) {
  b200::NvtxRange nvtx_range("b200_paged_prefill_fp8");
  int rc = check_attention(p);
  if (rc != B200_OK) return rc;
  if (p->num_seqs == 0 || p->num_tokens == 0) return B200_OK;
  if (!has_arrays(*p) || !p->cu_seqlens) return fail(B200_ERR_INVALID_ARGUMENT, "null pointer");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const PrefillPlan pl = prefill_plan(*p);
  if (pl.tensor_cores) {
    rc = check_workspace(workspace, workspace_bytes, pl.total);
    if (rc != B200_OK) return rc;
    return run_prefill(*p, pl, static_cast<char*>(workspace), st);
  }
  b200::AttnFp8Args a = attention_args(*p);
  a.cu_q = p->cu_seqlens;
  const cudaError_t e = b200::launch_row_fp8(a, p->dtype, p->num_tokens, st);
  if (e != cudaSuccess) return cuda_fail(e, "paged_prefill_fp8");
  return B200_OK;
}

}  // extern "C"
