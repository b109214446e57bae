// paged.h -- the paged KV cache as the kernels see it, and the launchers of the
// operators on it (rope.cu, paged_attn.cu, fa_packed.cu; entry points in
// paged_api.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/mlxcat_cuda.h"

namespace mlxcat {

// A cache of pages of 1 << page_shift tokens.  Element (page, head, token, d)
// sits at page * page_stride + head * head_stride + token * token_stride + d;
// key p of row r is token p & (page_size - 1) of page table[r][p >> page_shift].
struct PagedKV {
    void *k, *v;
    const int32_t *table;
    int64_t page_stride, head_stride, token_stride;
    int n_pages, page_shift, n_kv, D, rows, max_pages;
    int bf16;
};

// Codes that the paged kernels leave in *err.
enum PagedErr { PE_ROW = 51, PE_POS = 52, PE_PAGE = 53 };

// One past the last position a row's table can hold, kept far enough below 2^31
// that a tile's end still fits.
__host__ __device__ inline int paged_capacity(const PagedKV &kv) {
    const int64_t c = (int64_t)kv.max_pages << kv.page_shift;
    return c > 0x7fff0000 ? 0x7fff0000 : (int)c;
}

// Everything that these kernels read may be written by the kernel before, and they
// are launched early (programmatic serialisation): plain loads, since the read-only
// path (ld.global.nc) is for memory that nobody writes while the kernel lives, and
// neither griddepcontrol.wait nor an acquire orders it.
__device__ __forceinline__ int load_id(const int32_t *p) { return *p; }

struct RopeAppendArgs {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;   // elements between tokens
    int in_dtype, M, n_heads, with_rope;
    const float *q_norm, *k_norm;
    float eps;
    const int32_t *trow, *tpos;
    void *q_out;
    int32_t *err;
    int sm_count;
};
cudaError_t rope_append(const PagedKV &kv, const mlxcat_rope &rope, const RopeAppendArgs &a, cudaStream_t st);

// Queries of the decode / verify attention: M tokens in groups of qg tokens of
// one row; token m sees keys key_begin..tpos[m] of its row here.
struct PagedQuery {
    const void *q;
    int M, qg, n_heads;
    float scale_log2;
    const int32_t *trow, *tpos;
    void *out;
    int32_t *err;
};

// Partials of a shared-prefix pass: fp32 sums [splits][n_kv][D / 8][M * G rows][8]
// and (max, sum) pairs [splits][n_kv][M * G].  *ready: `token` (a new one each
// call) once the pass has waited for all that was launched before it, 0 again
// after the call.
struct PrefixPartials {
    float *o = nullptr, *ml = nullptr;
    unsigned long long *ready = nullptr, token = 0;
    int splits = 0, ctas = 0;   // CTAs of the pass
};

size_t paged_attn_scratch(int M, int qg, int n_heads, int n_kv, int D, int sm_count);
cudaError_t paged_attn(const PagedKV &kv, const PagedQuery &q, int key_begin, const PrefixPartials &pre, void *scratch,
                       int sm_count, cudaStream_t st);

// Attention on the 5th-generation tensor cores (fa_packed.cu).
struct PackedAttn {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;   // elements between tokens
    int bf16, Tq, Tk;
    const int32_t *cu_q, *cu_k;
    int n_seq, causal, n_heads, n_kv, D;
    float scale_log2;
    void *out;
    int32_t *err;
};
cudaError_t packed_attn(const PackedAttn &a, cudaStream_t st);

int prefix_items(int M, int n_heads, int n_kv);   // CTAs of the pass per split
int prefix_splits(int M, int n_heads, int n_kv, int prefix_len, int sm_count);
int prefix_max_splits(int M, int n_heads, int n_kv, int prefix_len, int sm_count);   // at most, on so many SMs or fewer
cudaError_t prefix_attn(const PagedKV &kv, const PagedQuery &q, int prefix_len, const PrefixPartials &part,
                        cudaStream_t st);

// message of the calling thread's last failed operator call (runtime.cu)
int op_error(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));

}  // namespace mlxcat
