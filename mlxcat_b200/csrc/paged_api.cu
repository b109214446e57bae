// paged_api.cu -- entry points of the paged-cache operators (include/mlxcat_cuda.h):
// checks of the arguments, then the launches of rope.cu, paged_attn.cu and
// fa_packed.cu.  Nothing is allocated, read back or kept between calls, but for the
// count of calls that fresh_token takes its values from.
#include <algorithm>
#include <atomic>
#include <chrono>
#include <cmath>

#include "../../include/mlxcat_cuda.h"
#include "kernels.h"
#include "paged.h"

using namespace mlxcat;

namespace {

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The cache's description as the kernels take it; false with a message when it
// does not describe one.
int paged_kv(const mlxcat_paged_kv *c, PagedKV *out) {
    if (!c || !c->k || !c->v || !c->page_table) return op_error(MLXCAT_E_INVALID, "paged cache: null pointer");
    if (c->dtype != MLXCAT_F16 && c->dtype != MLXCAT_BF16)
        return op_error(MLXCAT_E_INVALID, "paged cache: dtype %d (fp16 or bf16)", c->dtype);
    if (c->head_dim != 64 && c->head_dim != 128)
        return op_error(MLXCAT_E_INVALID, "paged cache: head_dim %d (64 or 128)", c->head_dim);
    if (c->page_size < 8 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)))
        return op_error(MLXCAT_E_INVALID, "paged cache: page_size %d (a power of two, 8..65536)", c->page_size);
    if (c->n_pages <= 0 || c->n_kv_heads <= 0 || c->rows <= 0 || c->max_pages <= 0)
        return op_error(MLXCAT_E_INVALID, "paged cache: empty shape");
    if (!aligned16(c->k) || !aligned16(c->v)) return op_error(MLXCAT_E_INVALID, "paged cache: k and v must be 16-byte aligned");
    // the three strides, innermost first: each must clear what lies inside it
    struct Dim {
        int64_t stride, count;
    } d[3] = {{c->token_stride, c->page_size}, {c->head_stride, c->n_kv_heads}, {c->page_stride, c->n_pages}};
    std::sort(d, d + 3, [](const Dim &x, const Dim &y) { return x.stride < y.stride; });
    int64_t extent = c->head_dim;
    for (const Dim &x : d) {
        if (x.stride <= 0 || x.stride % 8 || x.stride > ((int64_t)1 << 38))
            return op_error(MLXCAT_E_INVALID, "paged cache: strides must be positive multiples of 8 elements");
        if (x.count > 1 && x.stride < extent) return op_error(MLXCAT_E_INVALID, "paged cache: strides overlap");
        // extent + stride * (count - 1) <= 2^60, without a product that could wrap
        if (x.count > 1 && (((int64_t)1 << 60) - extent) / x.stride < x.count - 1)
            return op_error(MLXCAT_E_INVALID, "paged cache: extent too large");
        extent += x.stride * (x.count - 1);
    }
    PagedKV kv;
    kv.k = c->k; kv.v = c->v; kv.table = c->page_table;
    kv.page_stride = c->page_stride; kv.head_stride = c->head_stride; kv.token_stride = c->token_stride;
    kv.n_pages = c->n_pages;
    kv.page_shift = __builtin_ctz((unsigned)c->page_size);
    kv.n_kv = c->n_kv_heads; kv.D = c->head_dim; kv.rows = c->rows; kv.max_pages = c->max_pages;
    kv.bf16 = c->dtype == MLXCAT_BF16;
    *out = kv;
    return MLXCAT_OK;
}

// SM count of the current device, asked once per device
int sm_count() {
    static int n[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 0;
    int &x = n[dev & 63];
    if (!x) {
        int v = 0;
        if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
        x = v;
    }
    return x;
}
// The workspace queries work without a device: sized for the SMs of the B200.
constexpr int SM_MAX = 160;

float log2_scale(float scale, int D) { return (scale == 0.f ? 1.0f / sqrtf((float)D) : scale) * 1.4426950408889634f; }

bool attention_shape(int32_t M, int32_t qg, int32_t n_heads, int32_t n_kv, int32_t D) {
    return M > 0 && qg > 0 && n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && n_heads / n_kv <= 64 &&
           (D == 64 || D == 128) && (int64_t)M * n_heads <= ((int64_t)1 << 30) &&
           (int64_t)qg * (n_heads / n_kv) <= ((int64_t)1 << 24);
}

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

constexpr uintptr_t PARTIALS_ALIGN = 32;
struct PrefixLayout {
    int splits;
    size_t ml_at, ready_at, bytes;
};
PrefixLayout prefix_layout(int M, int n_heads, int n_kv, int D, int prefix_len) {
    PrefixLayout p;
    // the workspace is sized before the device is known
    p.splits = prefix_max_splits(M, n_heads, n_kv, prefix_len, SM_MAX);
    const size_t rows = (size_t)p.splits * M * n_heads;   // n_kv * (M * G)
    p.ml_at = up256(rows * D * 4);
    p.ready_at = p.ml_at + up256(rows * 8);
    // the pass stores its sums 32 bytes at a time: room to start on such a boundary in
    // a workspace that itself starts on one of 16
    p.bytes = p.ready_at + up256(sizeof(unsigned long long) + PARTIALS_ALIGN - 16);
    return p;
}

// What a shared-prefix call writes as its sign in the workspace: the workspace may
// hold anything, so 64 bits that no other call of this process writes and that
// stray contents match with probability 2^-64 (a bijection of a counter: the
// finaliser of SplitMix64, Steele, Lea and Flood, OOPSLA 2014).  Never 0.
unsigned long long fresh_token() {
    static const uint64_t seed = (uint64_t)std::chrono::steady_clock::now().time_since_epoch().count() << 20;
    static std::atomic<uint64_t> calls{0};
    for (;;) {
        uint64_t z = (seed + calls.fetch_add(1, std::memory_order_relaxed)) * 0x9E3779B97F4A7C15ull;
        z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
        z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
        z ^= z >> 31;
        if (z) return z;
    }
}

int query_of(const mlxcat_paged_kv *c, const void *q, int32_t M, int32_t qg, int32_t n_heads, float scale,
             const int32_t *trow, const int32_t *tpos, void *out, int32_t *err, PagedKV *kv, PagedQuery *pq) {
    const int rc = paged_kv(c, kv);
    if (rc != MLXCAT_OK) return rc;
    if (!q || !trow || !tpos || !out) return op_error(MLXCAT_E_INVALID, "paged attention: null pointer");
    if (!attention_shape(M, qg, n_heads, kv->n_kv, kv->D))
        return op_error(MLXCAT_E_INVALID, "paged attention: bad shape (M %d, qg %d, heads %d / %d)", M, qg, n_heads, kv->n_kv);
    if (!(scale >= 0.f) || std::isinf(scale)) return op_error(MLXCAT_E_INVALID, "paged attention: scale must be finite and not negative");
    if (!aligned16(q) || !aligned16(out)) return op_error(MLXCAT_E_INVALID, "paged attention: q and out must be 16-byte aligned");
    pq->q = q; pq->M = M; pq->qg = std::min(qg, M); pq->n_heads = n_heads; pq->scale_log2 = log2_scale(scale, kv->D);
    pq->trow = trow; pq->tpos = tpos; pq->out = out; pq->err = err;
    return MLXCAT_OK;
}

}  // namespace

extern "C" {

int mlxcat_rope_init(mlxcat_rope *rope, int32_t rotary_dim, int32_t layout, double theta,
                     const mlxcat_rope_scaling *s) {
    if (!rope || rotary_dim < 2 || rotary_dim > 256 || rotary_dim % 2 || !(theta > 1.0) || std::isinf(theta) ||
        (layout != MLXCAT_ROPE_HALF && layout != MLXCAT_ROPE_INTERLEAVED))
        return op_error(MLXCAT_E_INVALID, "rope: rotary_dim even in 2..256, layout half or interleaved, theta > 1");
    const int kind = s ? s->kind : MLXCAT_ROPE_SCALE_NONE;
    const double two_pi = 6.283185307179586476925286766559;
    if (kind < MLXCAT_ROPE_SCALE_NONE || kind > MLXCAT_ROPE_SCALE_YARN)
        return op_error(MLXCAT_E_INVALID, "rope: unknown scaling %d", kind);
    if (kind != MLXCAT_ROPE_SCALE_NONE && (!(s->factor >= 1.0) || std::isinf(s->factor)))
        return op_error(MLXCAT_E_INVALID, "rope: scaling factor must be at least 1");
    if (kind == MLXCAT_ROPE_SCALE_LLAMA3 &&
        (s->original_max_position <= 0 || !(s->low_freq_factor > 0.0) || !(s->high_freq_factor > s->low_freq_factor)))
        return op_error(MLXCAT_E_INVALID, "rope: original_max_position > 0 and 0 < low_freq_factor < high_freq_factor");
    if (kind == MLXCAT_ROPE_SCALE_YARN &&
        (s->original_max_position <= 0 || !(s->beta_slow > 0.0) || !(s->beta_fast > s->beta_slow) || !(s->mscale >= 0.0)))
        return op_error(MLXCAT_E_INVALID, "rope: original_max_position > 0, 0 < beta_slow < beta_fast, mscale >= 0");
    mlxcat_rope r = {};
    r.rotary_dim = rotary_dim;
    r.layout = layout;
    r.mscale = 1.f;
    double low = 0.0, high = 0.0;
    if (kind == MLXCAT_ROPE_SCALE_YARN) {
        // index of the pair that turns `rot` times within the original context
        auto at = [&](double rot) {
            return rotary_dim * std::log(s->original_max_position / (rot * two_pi)) / (2.0 * std::log(theta));
        };
        low = std::max(0.0, std::floor(at(s->beta_fast)));
        high = std::min(rotary_dim - 1.0, std::ceil(at(s->beta_slow)));
        r.mscale = (float)(s->mscale > 0.0 ? s->mscale : 0.1 * std::log(s->factor) + 1.0);
    }
    for (int i = 0; i < rotary_dim / 2; ++i) {
        double f = std::pow(theta, -2.0 * i / rotary_dim);
        if (kind == MLXCAT_ROPE_SCALE_LINEAR) f /= s->factor;
        if (kind == MLXCAT_ROPE_SCALE_LLAMA3) {
            const double n = s->original_max_position * f / two_pi;
            const double keep = std::min(1.0, std::max(0.0, (n - s->low_freq_factor) / (s->high_freq_factor - s->low_freq_factor)));
            f = (1.0 - keep) * f / s->factor + keep * f;
        }
        if (kind == MLXCAT_ROPE_SCALE_YARN) {
            const double ramp = std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 1e-3)));
            f = f / s->factor * ramp + f * (1.0 - ramp);
        }
        r.turns[i] = f / two_pi;
    }
    *rope = r;
    return MLXCAT_OK;
}

int mlxcat_op_rope_append(const mlxcat_paged_kv *c, const mlxcat_rope *rope, const void *q, const void *k, const void *v,
                          int32_t in_dtype, int64_t q_stride, int64_t k_stride, int64_t v_stride, int32_t M,
                          int32_t n_heads, const float *q_norm, const float *k_norm, float eps, const int32_t *trow,
                          const int32_t *tpos, void *q_out, int32_t *err, void *stream) {
    PagedKV kv;
    const int rc = paged_kv(c, &kv);
    if (rc != MLXCAT_OK) return rc;
    if (!k || !v || !trow || !tpos || !q != !q_out) return op_error(MLXCAT_E_INVALID, "rope append: null pointer");
    if (in_dtype != MLXCAT_F16 && in_dtype != MLXCAT_BF16 && in_dtype != MLXCAT_F32)
        return op_error(MLXCAT_E_INVALID, "rope append: unknown input type %d", in_dtype);
    if (M <= 0 || (q && n_heads <= 0) || (q && (int64_t)M * n_heads > ((int64_t)1 << 30)))
        return op_error(MLXCAT_E_INVALID, "rope append: bad shape (M %d, heads %d)", M, n_heads);
    if (!(eps >= 0.f)) return op_error(MLXCAT_E_INVALID, "rope append: eps must not be negative");
    if (rope && (rope->rotary_dim < 2 || rope->rotary_dim % 2 || rope->rotary_dim > kv.D ||
                 (rope->layout != MLXCAT_ROPE_HALF && rope->layout != MLXCAT_ROPE_INTERLEAVED)))
        return op_error(MLXCAT_E_INVALID, "rope append: rotary_dim %d does not fit head_dim %d", rope->rotary_dim, kv.D);
    const int64_t es = in_dtype == MLXCAT_F32 ? 4 : 2;
    const struct {
        const void *p;
        int64_t stride, heads;
    } in[3] = {{q, q_stride, n_heads}, {k, k_stride, kv.n_kv}, {v, v_stride, kv.n_kv}};
    for (const auto &x : in) {
        if (!x.p) continue;
        if (!aligned16(x.p) || x.stride % 8 || x.stride < x.heads * kv.D || x.stride > ((int64_t)1 << 30))
            return op_error(MLXCAT_E_INVALID, "rope append: inputs must be 16-byte aligned, token strides multiples of 8 that hold their heads");
        if (q_out) {
            const char *a0 = static_cast<const char *>(x.p), *a1 = a0 + ((M - 1) * x.stride + x.heads * kv.D) * es;
            const char *b0 = static_cast<const char *>(q_out), *b1 = b0 + (int64_t)M * n_heads * kv.D * 2;
            if (a0 < b1 && b0 < a1) return op_error(MLXCAT_E_INVALID, "rope append: q_out overlaps an input");
        }
    }
    if (q_out && !aligned16(q_out)) return op_error(MLXCAT_E_INVALID, "rope append: q_out must be 16-byte aligned");
    RopeAppendArgs a;
    a.q = q; a.k = k; a.v = v;
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
    a.in_dtype = in_dtype; a.M = M; a.n_heads = n_heads; a.with_rope = rope ? 1 : 0;
    a.q_norm = q_norm; a.k_norm = k_norm; a.eps = eps;
    a.trow = trow; a.tpos = tpos; a.q_out = q_out; a.err = err;
    a.sm_count = sm_count();
    if (a.sm_count <= 0) return op_error(MLXCAT_E_CUDA, "rope append: no CUDA device");
    const mlxcat_rope none = {};
    const cudaError_t e = rope_append(kv, rope ? *rope : none, a, (cudaStream_t)stream);
    if (e != cudaSuccess) return op_error(MLXCAT_E_CUDA, "rope append: %s", cudaGetErrorString(e));
    return MLXCAT_OK;
}

size_t mlxcat_op_paged_attention_workspace(int32_t M, int32_t qg, int32_t n_heads, int32_t n_kv, int32_t D) {
    if (!attention_shape(M, qg, n_heads, n_kv, D)) return 0;
    return up256(paged_attn_scratch(M, std::min(qg, M), n_heads, n_kv, D, SM_MAX));
}

int mlxcat_op_paged_attention(const mlxcat_paged_kv *c, const void *q, int32_t M, int32_t qg, int32_t n_heads,
                              float scale, const int32_t *trow, const int32_t *tpos, void *out, void *workspace,
                              size_t workspace_bytes, int32_t *err, void *stream) {
    return mlxcat_op_shared_prefix_attention(c, 0, q, M, qg, n_heads, scale, trow, tpos, out, workspace,
                                             workspace_bytes, err, stream);
}

size_t mlxcat_op_shared_prefix_attention_workspace(int32_t M, int32_t qg, int32_t n_heads, int32_t n_kv, int32_t D,
                                                   int32_t prefix_len) {
    const size_t own = mlxcat_op_paged_attention_workspace(M, qg, n_heads, n_kv, D);
    if (!own || prefix_len < 0) return 0;
    return own + (prefix_len ? prefix_layout(M, n_heads, n_kv, D, prefix_len).bytes : 0);
}

int mlxcat_op_shared_prefix_attention(const mlxcat_paged_kv *c, int32_t prefix_len, const void *q, int32_t M,
                                      int32_t qg, int32_t n_heads, float scale, const int32_t *trow,
                                      const int32_t *tpos, void *out, void *workspace, size_t workspace_bytes,
                                      int32_t *err, void *stream) {
    PagedKV kv;
    PagedQuery pq;
    const int rc = query_of(c, q, M, qg, n_heads, scale, trow, tpos, out, err, &kv, &pq);
    if (rc != MLXCAT_OK) return rc;
    if (prefix_len < 0 || prefix_len % c->page_size || prefix_len > paged_capacity(kv))
        return op_error(MLXCAT_E_INVALID, "shared prefix: %d keys are not whole pages of %d within the table", prefix_len, c->page_size);
    const size_t own = mlxcat_op_paged_attention_workspace(M, qg, n_heads, kv.n_kv, kv.D);
    const size_t need = mlxcat_op_shared_prefix_attention_workspace(M, qg, n_heads, kv.n_kv, kv.D, prefix_len);
    if (!workspace || workspace_bytes < need || !aligned16(workspace))
        return op_error(MLXCAT_E_INVALID, "paged attention: workspace of %zu bytes needed (16-byte aligned), %zu given", need, workspace_bytes);
    const int sms = sm_count();
    if (sms <= 0) return op_error(MLXCAT_E_CUDA, "paged attention: no CUDA device");
    PrefixPartials pre;
    const cudaStream_t st = (cudaStream_t)stream;
    // What the rows would read of the prefix one by one.  As long as that is about
    // what L2 holds they do, since the pass over the shared keys and the join of its
    // partials have a price of their own, which grows with the rows' own keys (they get
    // half the SMs).  8 KV heads of 128, row by row against once, 64 and 1,024 own keys:
    // 32 rows, 256 shared keys (34 MB) 14 and 31 us against 17 and 40; 32 rows, 1,024
    // keys (134 MB) 24 against 17 with 64 own keys; 64 rows, 1,024 keys (268 MB) 38 and
    // 63 against 21 and 62; 64 rows, 4,096 keys (1.1 GB) 111 against 27.
    const int64_t apart = (int64_t)((M + pq.qg - 1) / pq.qg) * prefix_len * kv.n_kv * kv.D * 4;
    if (apart <= ((int64_t)128 << 20)) prefix_len = 0;
    if (prefix_len) {
        const PrefixLayout l = prefix_layout(M, n_heads, kv.n_kv, kv.D, prefix_len);
        char *at = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(workspace) + own + PARTIALS_ALIGN - 1) & ~(PARTIALS_ALIGN - 1));
        pre.o = reinterpret_cast<float *>(at);
        pre.ml = reinterpret_cast<float *>(at + l.ml_at);
        pre.ready = reinterpret_cast<unsigned long long *>(at + l.ready_at);
        pre.token = fresh_token();
        pre.splits = std::min(l.splits, prefix_splits(M, n_heads, kv.n_kv, prefix_len, std::min(sms, SM_MAX)));
        pre.ctas = (int)std::min<int64_t>((int64_t)pre.splits * prefix_items(M, n_heads, kv.n_kv), 0x7fffffff);
        const cudaError_t e = prefix_attn(kv, pq, prefix_len, pre, st);
        if (e != cudaSuccess) return op_error(MLXCAT_E_CUDA, "shared prefix attention: %s", cudaGetErrorString(e));
    }
    const cudaError_t e = paged_attn(kv, pq, prefix_len, pre, workspace, std::min(sms, SM_MAX), st);
    if (e != cudaSuccess) return op_error(MLXCAT_E_CUDA, "paged attention: %s", cudaGetErrorString(e));
    return MLXCAT_OK;
}

int mlxcat_op_packed_attention(const void *q, const void *k, const void *v, int32_t dtype, int64_t q_stride,
                               int64_t k_stride, int64_t v_stride, int32_t Tq, int32_t Tk, const int32_t *cu_q,
                               const int32_t *cu_k, int32_t n_seq, int32_t causal, int32_t n_heads, int32_t n_kv,
                               int32_t D, float scale, void *out, int32_t *err, void *stream) {
    if (!q || !k || !v || !cu_q || !cu_k || !out) return op_error(MLXCAT_E_INVALID, "packed attention: null pointer");
    if (dtype != MLXCAT_F16 && dtype != MLXCAT_BF16)
        return op_error(MLXCAT_E_INVALID, "packed attention: dtype %d (fp16 or bf16)", dtype);
    if (Tq <= 0 || Tk <= 0 || n_seq <= 0 || !attention_shape(Tq, 1, n_heads, n_kv, D))
        return op_error(MLXCAT_E_INVALID, "packed attention: bad shape (Tq %d, Tk %d, sequences %d, heads %d / %d, head_dim %d)", Tq,
                        Tk, n_seq, n_heads, n_kv, D);
    if (!(scale >= 0.f) || std::isinf(scale)) return op_error(MLXCAT_E_INVALID, "packed attention: scale must be finite and not negative");
    const struct {
        const void *p;
        int64_t stride;
        int heads;
    } in[4] = {{q, q_stride, n_heads}, {k, k_stride, n_kv}, {v, v_stride, n_kv}, {out, (int64_t)n_heads * D, n_heads}};
    for (const auto &x : in)
        if (!aligned16(x.p) || x.stride % 8 || x.stride < (int64_t)x.heads * D || x.stride > ((int64_t)1 << 38))
            return op_error(MLXCAT_E_INVALID, "packed attention: buffers must be 16-byte aligned, token strides multiples of 8 that hold their heads");
    PackedAttn a;
    a.q = q; a.k = k; a.v = v;
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride;
    a.bf16 = dtype == MLXCAT_BF16; a.Tq = Tq; a.Tk = Tk; a.cu_q = cu_q; a.cu_k = cu_k; a.n_seq = n_seq;
    a.causal = causal ? 1 : 0; a.n_heads = n_heads; a.n_kv = n_kv; a.D = D;
    a.scale_log2 = log2_scale(scale, D); a.out = out; a.err = err;
    const cudaError_t e = packed_attn(a, (cudaStream_t)stream);
    if (e != cudaSuccess) return op_error(MLXCAT_E_CUDA, "packed attention: %s", cudaGetErrorString(e));
    return MLXCAT_OK;
}

}  // extern "C"
