// C ABI of the serving operators (paged K/V cache, token scores): argument
// checks and the launchers' arguments.  Declared in include/slr_b200.h.
#include <cmath>
#include <string>

#include "internal.hpp"

using namespace slr;

namespace {

int check_cache(const slr_kv_cache* c) {
  if (!c) return fail(SLR_ERR_INVALID_ARGUMENT, "cache is NULL");
  if (c->dtype != SLR_F32 && c->dtype != SLR_F16 && c->dtype != SLR_BF16)
    return fail(SLR_ERR_UNSUPPORTED_DTYPE, "kv cache: dtype must be float32/float16/bfloat16");
  if (c->num_layers < 1 || c->num_pages < 1 || c->kv_heads < 1 || c->max_rows < 1 || c->max_pages < 1)
    return fail(SLR_ERR_INVALID_ARGUMENT, "kv cache: num_layers, num_pages, kv_heads, max_rows and max_pages must be >= 1");
  if (c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8)
    return fail(SLR_ERR_INVALID_ARGUMENT, "kv cache: head_dim must be a multiple of 8 up to 256");
  if (c->page_size < 16 || c->page_size > 1024 || c->page_size % 16)
    return fail(SLR_ERR_INVALID_ARGUMENT, "kv cache: page_size must be a multiple of 16 up to 1024");
  if (c->max_rows > SLR_KV_MAX_ROWS)
    return fail(SLR_ERR_INVALID_ARGUMENT, "kv cache: max_rows must be at most " + std::to_string(SLR_KV_MAX_ROWS));
  if (int64_t(c->max_pages) * c->page_size >= (int64_t(1) << 31))
    return fail(SLR_ERR_INVALID_ARGUMENT, "kv cache: max_pages * page_size must be below 2^31");
  const int64_t e = int64_t(dtype_size(c->dtype));
  for (int64_t s : {c->layer_stride, c->page_stride, c->head_stride, c->token_stride})
    if (s < 0 || s * e % 16) return fail(SLR_ERR_INVALID_ARGUMENT, "kv cache: strides must be multiples of 16 bytes");
  // the block of one page: heads and slots in either order, without gaps
  const bool by_head = c->token_stride == c->head_dim && c->head_stride == int64_t(c->page_size) * c->head_dim;
  const bool by_token = c->head_stride == c->head_dim && c->token_stride == int64_t(c->kv_heads) * c->head_dim;
  if (!by_head && !by_token) return fail(SLR_ERR_INVALID_ARGUMENT, "kv cache: the block of a page must be contiguous");
  if (c->page_stride < int64_t(c->kv_heads) * c->page_size * c->head_dim)
    return fail(SLR_ERR_INVALID_ARGUMENT, "kv cache: pages overlap");
  return SLR_OK;
}

// check_cache, and the pointers that a launch reads
int check_launch(const slr_kv_cache* c) {
  int rc = check_cache(c);
  if (rc) return rc;
  if (!c->k || !c->v || !c->state) return fail(SLR_ERR_INVALID_ARGUMENT, "kv cache: k, v or state is NULL");
  if (!aligned16(c->k) || !aligned16(c->v))
    return fail(SLR_ERR_INVALID_ARGUMENT, "kv cache: k and v must be 16-byte aligned");
  return SLR_OK;
}

int check_workspace(const void* ws, size_t have, size_t need) {
  if (!ws) return fail(SLR_ERR_WORKSPACE, "workspace is NULL");
  if (have < need) return fail(SLR_ERR_WORKSPACE, "workspace too small: need " + std::to_string(need) + " bytes");
  if (reinterpret_cast<uintptr_t>(ws) & 255u) return fail(SLR_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  return SLR_OK;
}

PagesArgs pages_args(const slr_kv_cache& c, void* ws) {
  const int64_t e = int64_t(dtype_size(c.dtype));
  PagesArgs p;
  p.state = c.state;
  p.rows = c.max_rows;
  p.num_pages = c.num_pages;
  p.max_pages = c.max_pages;
  p.page_size = c.page_size;
  p.k = static_cast<uint8_t*>(c.k);
  p.v = static_cast<uint8_t*>(c.v);
  p.layer_bytes = c.layer_stride * e;
  p.page_stride_bytes = c.page_stride * e;
  p.page_bytes = int64_t(c.kv_heads) * c.page_size * c.head_dim * e;
  p.layers = c.num_layers;
  p.workspace = ws;
  return p;
}

int32_t* lens_of(const slr_kv_cache& c) { return c.state + SLR_KV_HEADER_WORDS; }
int32_t* table_of(const slr_kv_cache& c) { return lens_of(c) + c.max_rows + c.num_pages; }

const void* layer_base(const slr_kv_cache& c, const void* base, int layer) {
  return static_cast<const uint8_t*>(base) + int64_t(layer) * c.layer_stride * int64_t(dtype_size(c.dtype));
}

}  // namespace

extern "C" {

size_t slr_kv_pages_workspace_size(const slr_kv_cache* cache) {
  if (check_cache(cache)) return 0;
  return kv_pages_workspace_size(cache->max_rows, cache->num_pages);
}

size_t slr_kv_attend_workspace_size(const slr_kv_cache* cache, int32_t rows, int32_t heads) {
  if (check_cache(cache)) return 0;
  if (rows < 0 || rows > cache->max_rows || heads < 1 || heads % cache->kv_heads) {
    fail(SLR_ERR_INVALID_ARGUMENT, "kv attend: rows out of range, or heads not a multiple of kv_heads");
    return 0;
  }
  size_t n = 0;
  const int64_t longest = int64_t(cache->max_pages) * cache->page_size;
  return attend_workspace_size(cache->dtype, cache->head_dim, rows, cache->kv_heads, heads / cache->kv_heads, longest, &n)
             ? 0
             : n;
}

int slr_kv_advance(const slr_kv_cache* cache, const int32_t* parents, const int32_t* n_new, int32_t n_all,
                   void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_launch(cache);
  if (!rc) rc = check_workspace(workspace, workspace_bytes, kv_pages_workspace_size(cache->max_rows, cache->num_pages));
  if (rc) return rc;
  return launch_kv_advance(pages_args(*cache, workspace), n_new, n_all, parents, static_cast<cudaStream_t>(stream));
}

int slr_kv_compact(const slr_kv_cache* cache, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_launch(cache);
  if (!rc) rc = check_workspace(workspace, workspace_bytes, kv_pages_workspace_size(cache->max_rows, cache->num_pages));
  if (rc) return rc;
  return launch_kv_compact(pages_args(*cache, workspace), static_cast<cudaStream_t>(stream));
}

int slr_kv_copy_pages(const slr_kv_cache* cache, const int32_t* src, const int32_t* dst, int32_t n, void* stream) {
  int rc = check_launch(cache);
  if (rc) return rc;
  if (n < 0 || (n > 0 && (!src || !dst))) return fail(SLR_ERR_INVALID_ARGUMENT, "kv copy: bad page lists");
  if (n == 0) return SLR_OK;
  return launch_kv_copy(pages_args(*cache, nullptr), src, dst, n, static_cast<cudaStream_t>(stream));
}

int slr_kv_append(const slr_kv_cache* cache, int32_t layer, const void* k, int64_t k_row_stride,
                  int64_t k_head_stride, const void* v, int64_t v_row_stride, int64_t v_head_stride, int64_t tokens,
                  const int32_t* cu_tokens, void* stream) {
  int rc = check_launch(cache);
  if (rc) return rc;
  if (layer < 0 || layer >= cache->num_layers) return fail(SLR_ERR_INVALID_ARGUMENT, "kv append: layer out of range");
  if (tokens < 0 || tokens >= (int64_t(1) << 31) || (!cu_tokens && tokens > cache->max_rows))
    return fail(SLR_ERR_INVALID_ARGUMENT, "kv append: tokens out of range (one per row without cu_tokens)");
  if (k_row_stride < 0 || k_head_stride < 0 || v_row_stride < 0 || v_head_stride < 0)
    return fail(SLR_ERR_INVALID_ARGUMENT, "kv append: strides must be >= 0");
  if (tokens == 0) return SLR_OK;
  if (!k || !v) return fail(SLR_ERR_INVALID_ARGUMENT, "kv append: k or v is NULL");
  AppendArgs a;
  a.k = const_cast<void*>(layer_base(*cache, cache->k, layer));
  a.v = const_cast<void*>(layer_base(*cache, cache->v, layer));
  a.page_stride = cache->page_stride;
  a.head_stride = cache->head_stride;
  a.token_stride = cache->token_stride;
  a.table = table_of(*cache);
  a.lens = lens_of(*cache);
  a.new_k = k;
  a.new_v = v;
  a.k_row = k_row_stride;
  a.k_head = k_head_stride;
  a.v_row = v_row_stride;
  a.v_head = v_head_stride;
  a.cu = cu_tokens;
  a.tokens = tokens;
  a.rows = cache->max_rows;
  a.kv_heads = cache->kv_heads;
  a.dim = cache->head_dim;
  a.page_size = cache->page_size;
  a.max_pages = cache->max_pages;
  a.num_pages = cache->num_pages;
  a.dtype = cache->dtype;
  return launch_kv_append(a, static_cast<cudaStream_t>(stream));
}

int slr_kv_attend(const slr_kv_cache* cache, int32_t layer, const void* q, int64_t q_row_stride,
                  int64_t q_head_stride, void* out, int64_t o_row_stride, int64_t o_head_stride, float* lse,
                  int32_t rows, int32_t heads, float scale, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_launch(cache);
  if (rc) return rc;
  if (layer < 0 || layer >= cache->num_layers) return fail(SLR_ERR_INVALID_ARGUMENT, "kv attend: layer out of range");
  if (rows < 0 || rows > cache->max_rows) return fail(SLR_ERR_INVALID_ARGUMENT, "kv attend: rows out of range");
  if (heads < 1 || heads % cache->kv_heads)
    return fail(SLR_ERR_INVALID_ARGUMENT, "kv attend: heads must be a multiple of kv_heads");
  if (heads > 4096) return fail(SLR_ERR_INVALID_ARGUMENT, "kv attend: at most 4096 heads");
  if (q_row_stride < 0 || q_head_stride < 0 || o_row_stride < 0 || o_head_stride < 0)
    return fail(SLR_ERR_INVALID_ARGUMENT, "kv attend: strides must be >= 0");
  if (!std::isfinite(scale)) return fail(SLR_ERR_INVALID_ARGUMENT, "kv attend: scale must be finite");
  // the list of tiles (8 tokens or more each, 3 places behind each row's) is counted in 32 bits
  if (int64_t(cache->max_rows) * (int64_t(cache->max_pages) * cache->page_size / 8 + 4) >= (int64_t(1) << 31))
    return fail(SLR_ERR_UNSUPPORTED, "kv attend: max_rows * max_pages * page_size must be below about 2^34");
  if (rows == 0) return SLR_OK;
  if (!q || !out) return fail(SLR_ERR_INVALID_ARGUMENT, "kv attend: q or out is NULL");
  if (reinterpret_cast<uintptr_t>(workspace) & 255u) return fail(SLR_ERR_WORKSPACE, "workspace must be 256-byte aligned");
  // every output vector has its own place: the heads within a row's stride, or the rows within a head's
  auto apart = [&](int64_t n_in, int64_t in, int64_t n_out, int64_t outer) {
    if (n_in > 1 && in < cache->head_dim) return false;
    const __int128 span = (n_in > 1 ? __int128(in) * (n_in - 1) : 0) + cache->head_dim;
    return n_out <= 1 || outer >= span;
  };
  if (!apart(heads, o_head_stride, rows, o_row_stride) && !apart(rows, o_row_stride, heads, o_head_stride))
    return fail(SLR_ERR_INVALID_ARGUMENT, "kv attend: out overlaps itself");
  AttendArgs a;
  a.k = layer_base(*cache, cache->k, layer);
  a.v = layer_base(*cache, cache->v, layer);
  a.page_stride = cache->page_stride;
  a.head_stride = cache->head_stride;
  a.token_stride = cache->token_stride;
  a.table = table_of(*cache);
  a.lens = lens_of(*cache);
  a.q = q;
  a.q_row = q_row_stride;
  a.q_head = q_head_stride;
  a.out = out;
  a.o_row = o_row_stride;
  a.o_head = o_head_stride;
  a.lse = lse;
  a.rows = rows;
  a.heads = heads;
  a.kv_heads = cache->kv_heads;
  a.dim = cache->head_dim;
  a.page_size = cache->page_size;
  a.max_pages = cache->max_pages;
  a.num_pages = cache->num_pages;
  a.scale = scale;
  a.dtype = cache->dtype;
  a.workspace = workspace;
  a.workspace_bytes = workspace_bytes;
  return launch_attend(a, static_cast<cudaStream_t>(stream));
}

int slr_token_logprobs(const void* logits, int64_t row_stride, int64_t rows, int64_t vocab, int dtype,
                       const int64_t* targets, float* logprob, float* entropy, int32_t top, int64_t* top_ids,
                       float* top_logprobs, void* stream) {
  if (dtype != SLR_F32 && dtype != SLR_F16 && dtype != SLR_BF16)
    return fail(SLR_ERR_UNSUPPORTED_DTYPE, "token logprobs: dtype must be float32/float16/bfloat16");
  if (rows < 0 || vocab < 1 || vocab >= (int64_t(1) << 31))
    return fail(SLR_ERR_INVALID_ARGUMENT, "token logprobs: rows must be >= 0 and vocab in [1, 2^31)");
  if (rows > (int64_t(1) << 27)) return fail(SLR_ERR_INVALID_ARGUMENT, "token logprobs: at most 2^27 rows");
  if (row_stride == 0) row_stride = vocab;
  if (row_stride < 0) return fail(SLR_ERR_INVALID_ARGUMENT, "token logprobs: row_stride must be >= 0");
  if (top < 0 || top > SLR_MAX_TOP || top > vocab)
    return fail(SLR_ERR_INVALID_ARGUMENT, "token logprobs: top must be in [0, min(32, vocab)]");
  if ((targets == nullptr) != (logprob == nullptr))
    return fail(SLR_ERR_INVALID_ARGUMENT, "token logprobs: targets and logprob go together");
  if (rows == 0) return SLR_OK;
  if (!logits || (top && (!top_ids || !top_logprobs)))
    return fail(SLR_ERR_INVALID_ARGUMENT, "token logprobs: null tensor pointer");
  LogprobArgs a;
  a.logits = logits;
  a.row_stride = row_stride;
  a.rows = rows;
  a.vocab = vocab;
  a.dtype = dtype;
  a.targets = targets;
  a.logprob = logprob;
  a.entropy = entropy;
  a.top = top;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  return launch_logprobs(a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
