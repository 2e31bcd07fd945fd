// C-ABI entry points of the operators on a paged cache and of rotary positions (see include/splitd_attn.h): argument
// checks, then the launch. Everything that is checked here needs no device value.
#include <cstring>

#include "../../include/splitd_attn.h"
#include "launch.cuh"

namespace sd {

namespace {

int check_heads(int heads_q, int heads_kv, int head_dim, int dtype) {
  if (head_dim != kHeadDim) return fail(SPLITD_ERR_INVALID_ARGUMENT, "head_dim == 512 is required, got %d", head_dim);
  if (heads_q <= 0 || heads_kv <= 0 || heads_q % heads_kv != 0)
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "heads_q (%d) must be a positive multiple of heads_kv (%d)", heads_q, heads_kv);
  if (dtype != SPLITD_DTYPE_BF16 && dtype != SPLITD_DTYPE_FP16)
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "dtype must be SPLITD_DTYPE_BF16 or SPLITD_DTYPE_FP16");
  return 0;
}

int check_rows(const void* base, const int64_t* strides, int first, const char* what) {
  if (reinterpret_cast<uintptr_t>(base) % 16 != 0)
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "%s: base pointer must be 16-byte aligned", what);
  for (int i = first; i < 3; ++i)
    if (strides[i] % 8 != 0)
      return fail(SPLITD_ERR_INVALID_ARGUMENT, "%s: stride %lld of dim %d must be a multiple of 8 elements", what,
                  (long long)strides[i], i);
  return 0;
}

int check_pages(int batch, int num_pages, int page_size, int max_pages) {
  // the batch is a grid dimension of some kernels
  if (batch <= 0 || batch > 65535) return fail(SPLITD_ERR_INVALID_ARGUMENT, "batch must be in 1 .. 65535, got %d", batch);
  if (num_pages < 0 || page_size <= 0 || max_pages < 0)
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "num_pages, page_size (> 0) and max_pages must not be negative");
  return 0;
}

int check_rotary(const double* inv_freq, int rotary_dim) {
  if (rotary_dim < 0 || rotary_dim > kHeadDim || rotary_dim % 2 != 0)
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "rotary_dim must be even and in 0 .. 512, got %d", rotary_dim);
  if (rotary_dim > 0 && !inv_freq) return fail(SPLITD_ERR_INVALID_ARGUMENT, "inv_freq must not be NULL");
  return 0;
}

}  // namespace

}  // namespace sd

using namespace sd;

extern "C" {

size_t splitd_paged_attn_workspace_bytes(const splitd_paged_params* p) { return p ? paged_workspace_bytes(p) : 0; }

int splitd_paged_attn(const splitd_paged_params* p, void* stream) {
  clear_error();
  if (!p) return fail(SPLITD_ERR_INVALID_ARGUMENT, "params is NULL");
  if (!p->q || !p->k_pages || !p->v_pages || !p->o || !p->page_table || !p->seqlens_k)
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "q, k_pages, v_pages, o, page_table and seqlens_k must not be NULL");
  if (int e = check_heads(p->heads_q, p->heads_kv, p->head_dim, p->dtype)) return e;
  if (int e = check_pages(p->batch, p->num_pages, p->page_size, p->max_pages)) return e;
  if (p->seqlen_q <= 0) return fail(SPLITD_ERR_INVALID_ARGUMENT, "seqlen_q must be > 0");
  if (static_cast<int64_t>(p->seqlen_q) * p->heads_q > (1 << 24))
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "seqlen_q * heads_q must be at most 2^24: this is the form for a few query tokens");
  if (!(p->softmax_scale > 0.f)) return fail(SPLITD_ERR_INVALID_ARGUMENT, "softmax_scale must be > 0");
  if (!(p->softcap >= 0.f)) return fail(SPLITD_ERR_INVALID_ARGUMENT, "softcap must be >= 0");
  if (p->local && (p->window_left < -1 || p->window_right < -1))
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "window_left / window_right must be >= -1");
  if (p->causal && p->local)
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "causal and a sliding window are mutually exclusive");
  if (p->key_weights && p->key_weights_len <= 0)
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "key_weights needs key_weights_len > 0");
  if (int e = check_rows(p->q, p->q_strides, 0, "q")) return e;
  if (int e = check_rows(p->o, p->o_strides, 0, "o")) return e;
  if (int e = check_rows(p->k_pages, p->k_strides, 0, "k_pages")) return e;
  if (int e = check_rows(p->v_pages, p->v_strides, 0, "v_pages")) return e;
  const size_t need = paged_workspace_bytes(p);
  if (!p->workspace || p->workspace_bytes < need || reinterpret_cast<uintptr_t>(p->workspace) % 256 != 0)
    return fail(SPLITD_ERR_WORKSPACE, "workspace: %zu bytes, 256-byte aligned, required, got %zu", need, p->workspace_bytes);
  if (int e = check_device()) return e;
  return launch_paged_attn(p, static_cast<cudaStream_t>(stream));
}

int splitd_rotary(const splitd_rotary_params* p, void* stream) {
  clear_error();
  if (!p) return fail(SPLITD_ERR_INVALID_ARGUMENT, "params is NULL");
  if (!p->q && !p->k) return fail(SPLITD_ERR_INVALID_ARGUMENT, "q and k must not both be NULL");
  if ((p->q && !p->q_out) || (p->k && !p->k_out)) return fail(SPLITD_ERR_INVALID_ARGUMENT, "an input without its output");
  if (!p->positions) return fail(SPLITD_ERR_INVALID_ARGUMENT, "positions must not be NULL");
  // the two are turned side by side: neither number of heads has to divide the other
  if (int e = check_heads(p->q ? p->heads_q : 1, 1, p->head_dim, p->dtype)) return e;
  if (int e = check_heads(p->k ? p->heads_kv : 1, 1, p->head_dim, p->dtype)) return e;
  if (p->batch <= 0 || p->seqlen <= 0) return fail(SPLITD_ERR_INVALID_ARGUMENT, "batch and seqlen must be > 0");
  if (int e = check_rotary(p->inv_freq, p->rotary_dim)) return e;
  if (p->q) {
    if (int e = check_rows(p->q, p->q_strides, 0, "q")) return e;
    if (int e = check_rows(p->q_out, p->q_out_strides, 0, "q_out")) return e;
  }
  if (p->k) {
    if (int e = check_rows(p->k, p->k_strides, 0, "k")) return e;
    if (int e = check_rows(p->k_out, p->k_out_strides, 0, "k_out")) return e;
  }
  if (int e = check_device()) return e;
  return launch_rotary(p, static_cast<cudaStream_t>(stream));
}

int splitd_paged_append(const splitd_append_params* p, void* stream) {
  clear_error();
  if (!p) return fail(SPLITD_ERR_INVALID_ARGUMENT, "params is NULL");
  if (!p->k || !p->v || !p->k_pages || !p->v_pages || !p->page_table || !p->seqlens_k)
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "k, v, k_pages, v_pages, page_table and seqlens_k must not be NULL");
  if (p->q && !p->q_out) return fail(SPLITD_ERR_INVALID_ARGUMENT, "q without q_out");
  if (int e = check_heads(p->q ? p->heads_q : p->heads_kv, p->heads_kv, p->head_dim, p->dtype)) return e;
  if (int e = check_pages(p->batch, p->num_pages, p->page_size, p->max_pages)) return e;
  if (p->cu_seqlens ? p->total_tokens <= 0 : p->seqlen <= 0)
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "there must be at least one new token");
  if (int e = check_rotary(p->inv_freq, p->inv_freq ? p->rotary_dim : 0)) return e;
  const int first = p->cu_seqlens ? 1 : 0;
  if (p->q) {
    if (int e = check_rows(p->q, p->q_strides, first, "q")) return e;
    if (int e = check_rows(p->q_out, p->q_out_strides, first, "q_out")) return e;
  }
  if (int e = check_rows(p->k, p->k_strides, first, "k")) return e;
  if (int e = check_rows(p->v, p->v_strides, first, "v")) return e;
  if (int e = check_rows(p->k_pages, p->k_page_strides, 0, "k_pages")) return e;
  if (int e = check_rows(p->v_pages, p->v_page_strides, 0, "v_pages")) return e;
  if (int e = check_device()) return e;
  return launch_paged_append(p, static_cast<cudaStream_t>(stream));
}

int splitd_paged_evict(const splitd_evict_params* p, void* stream) {
  clear_error();
  if (!p) return fail(SPLITD_ERR_INVALID_ARGUMENT, "params is NULL");
  if (!p->k_pages || !p->v_pages || !p->page_table || !p->new_page_table || !p->seqlens_k || !p->key_weights ||
      !p->new_seqlens || !p->kept || !p->new_weights)
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "a tensor is NULL");
  if (int e = check_heads(p->heads_kv, p->heads_kv, p->head_dim, SPLITD_DTYPE_BF16)) return e;
  if (int e = check_pages(p->batch, p->num_pages, p->page_size, p->max_pages)) return e;
  if (p->keep > 1 << 30) return fail(SPLITD_ERR_INVALID_ARGUMENT, "keep must be at most 2^30, got %d", p->keep);
  if (p->keep <= 0 || p->keep_first < 0 || p->keep_recent < 0 ||
      static_cast<int64_t>(p->keep_first) + p->keep_recent > p->keep)
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "keep must be > 0 and at least keep_first + keep_recent, got %d, %d, %d", p->keep,
                p->keep_first, p->keep_recent);
  if (p->new_max_pages < 0 || static_cast<int64_t>(p->new_max_pages) * p->page_size < p->keep)
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "new_page_table: %d pages of %d slots do not hold %d", p->new_max_pages, p->page_size,
                p->keep);
  if (p->new_weights_len != 0 && (p->new_weights_len < p->keep || p->new_weights_len > 1 << 30))
    return fail(SPLITD_ERR_INVALID_ARGUMENT, "new_weights_len (%d) must be 0, or at least keep (%d) and at most 2^30",
                p->new_weights_len, p->keep);
  if (p->key_weights_len < 0) return fail(SPLITD_ERR_INVALID_ARGUMENT, "key_weights_len must not be negative");
  if (int e = check_rows(p->k_pages, p->k_strides, 0, "k_pages")) return e;
  if (int e = check_rows(p->v_pages, p->v_strides, 0, "v_pages")) return e;
  if (int e = check_device()) return e;
  return launch_evict(p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
