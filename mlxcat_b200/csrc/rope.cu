// rope.cu -- per-head RMSNorm of queries and keys, rotary positions, and the
// append of keys and values to a paged cache, in one pass over the projection's
// output.
//
//   y = x * w / sqrt(mean(x^2) + eps)             (q and k heads, optional)
//   (a, b) -> s (a cos t - b sin t, b cos t + a sin t),  t = pos * f_i
//
// for the pairs (i, i + r/2) (half layout) or (2i, 2i + 1) (interleaved) of the
// first r features; the others pass through.  The angle is formed in 64 bits as
// turns (pos * f_i / 2 pi, the integer part dropped), so a position of 2^31
// still has its fraction to 2^-22 of a turn; only the fraction goes to fp32.
//
// Bound by HBM: every input is read and every output written once.  One CTA per
// token: its r/2 angles are computed once for all its heads.  A thread owns 8
// consecutive features (16-byte stores); a head is D/8 neighbouring lanes, so
// the sum of squares and the rotation partner of the half layout are shuffles.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace mlxcat {

namespace {

constexpr int RA_THREADS = 256;

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename TI>
__device__ __forceinline__ void load8(const TI *p, float *x) {
    constexpr int W = sizeof(TI) / 2;   // 16-byte words per 8 elements
    __align__(16) TI v[8];
#pragma unroll
    for (int i = 0; i < W; ++i) reinterpret_cast<uint4 *>(v)[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f<TI>(v[i]);
}

template <typename TI, typename TO, int D>
__global__ void __launch_bounds__(RA_THREADS)
rope_append_kernel(const PagedKV kv, const __grid_constant__ mlxcat_rope rope, const RopeAppendArgs a) {
    constexpr int LPH = D / 8;   // lanes per head
    __shared__ float2 cs[D / 2];
    griddep_launch_dependents();
    griddep_wait();
    const int m = blockIdx.x;
    const int row = __ldg(a.trow + m), pos = __ldg(a.tpos + m);
    if (row < 0) return;   // padding
    const int half = a.with_rope ? rope.rotary_dim / 2 : 0;
    for (int i = threadIdx.x; i < half; i += RA_THREADS) {
        const double turns = (double)pos * rope.turns[i];
        float s, c;
        sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
        cs[i] = make_float2(c * rope.mscale, s * rope.mscale);
    }
    // the token's slot; one outside the table or the cache is not written
    int page = -1;
    int bad = 0;
    if (row >= kv.rows) bad = PE_ROW;
    else if (pos < 0 || pos >= paged_capacity(kv)) bad = PE_POS;
    else {
        page = __ldg(kv.table + (size_t)row * kv.max_pages + (pos >> kv.page_shift));
        if (page < 0 || page >= kv.n_pages) { bad = PE_PAGE; page = -1; }
    }
    if (bad && threadIdx.x == 0 && a.err) atomicExch(a.err, bad);
    const int64_t slot = page < 0 ? 0 : (int64_t)page * kv.page_stride +
                                            (int64_t)(pos & ((1 << kv.page_shift) - 1)) * kv.token_stride;
    __syncthreads();
    const int nq = a.q ? a.n_heads : 0, heads = nq + 2 * kv.n_kv;
    const int vecs = heads * LPH;
    const bool inter = rope.layout == MLXCAT_ROPE_INTERLEAVED;
    for (int v0 = threadIdx.x & ~31; v0 < vecs; v0 += RA_THREADS) {   // warp-uniform bound: every lane shuffles
        const int vi = v0 + (threadIdx.x & 31);
        const bool on = vi < vecs;
        const int hh = (on ? vi : vecs - 1) / LPH, j = (on ? vi : vecs - 1) % LPH, d0 = j * 8;
        const bool is_q = hh < nq, is_v = hh >= nq + kv.n_kv;
        const int hl = is_q ? hh : is_v ? hh - nq - kv.n_kv : hh - nq;
        const TI *src = reinterpret_cast<const TI *>(is_q ? a.q : is_v ? a.v : a.k) +
                        (int64_t)m * (is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride) + (int64_t)hl * D;
        float x[8];
        load8<TI>(src + d0, x);
        const float *w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        float r = 1.f;
        if (w) {
            r = 1.0f / sqrtf(ss / (float)D + a.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * r * __ldg(w + d0 + i);
        }
        if (half) {
            if (inter) {
                if (!is_v) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2)
                        if (d0 + i < 2 * half) {
                            const float2 t = cs[(d0 + i) >> 1];
                            const float p = x[i], q = x[i + 1];
                            x[i] = p * t.x - q * t.y;
                            x[i + 1] = q * t.x + p * t.y;
                        }
                }
            } else if ((half & 7) == 0) {
                // partner vector: half/8 lanes on or back, same register
                const int hv = half >> 3;
                const bool lo = j < hv, in = j < 2 * hv;
                const int lane = threadIdx.x & 31, from = in ? (lo ? lane + hv : lane - hv) : lane;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float o = __shfl_sync(0xffffffffu, x[i], from);
                    if (in && !is_v) {
                        const float2 t = cs[lo ? d0 + i : d0 + i - half];
                        x[i] = lo ? x[i] * t.x - o * t.y : x[i] * t.x + o * t.y;
                    }
                }
            } else if (!is_v) {
                // a rotary width whose half is no multiple of 8: the partner is read again
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int d = d0 + i;
                    if (d >= 2 * half) continue;
                    const int e = d < half ? d + half : d - half;
                    float o = to_f<TI>(src[e]);
                    if (w) o = o * r * __ldg(w + e);
                    const float2 t = cs[d < half ? d : e];
                    x[i] = d < half ? x[i] * t.x - o * t.y : x[i] * t.x + o * t.y;
                }
            }
        }
        if (!on) continue;
        __align__(16) TO y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = from_f<TO>(x[i]);
        TO *dst = nullptr;
        if (is_q) dst = reinterpret_cast<TO *>(a.q_out) + ((size_t)m * a.n_heads + hl) * D;
        else if (page >= 0) dst = reinterpret_cast<TO *>(is_v ? kv.v : kv.k) + slot + (int64_t)hl * kv.head_stride;
        if (dst) *reinterpret_cast<uint4 *>(dst + d0) = *reinterpret_cast<const uint4 *>(y);
    }
}

template <typename TI, typename TO>
cudaError_t launch_d(const PagedKV &kv, const mlxcat_rope &rope, const RopeAppendArgs &a, cudaStream_t st) {
    if (kv.D == 128)
        return launch_pdl(rope_append_kernel<TI, TO, 128>, dim3(a.M), dim3(RA_THREADS), 0, st, kv, rope, a);
    return launch_pdl(rope_append_kernel<TI, TO, 64>, dim3(a.M), dim3(RA_THREADS), 0, st, kv, rope, a);
}

template <typename TI>
cudaError_t launch_o(const PagedKV &kv, const mlxcat_rope &rope, const RopeAppendArgs &a, cudaStream_t st) {
    return kv.bf16 ? launch_d<TI, __nv_bfloat16>(kv, rope, a, st) : launch_d<TI, __half>(kv, rope, a, st);
}

}  // namespace

cudaError_t rope_append(const PagedKV &kv, const mlxcat_rope &rope, const RopeAppendArgs &a, cudaStream_t st) {
    switch (a.in_dtype) {
        case MLXCAT_F32: return launch_o<float>(kv, rope, a, st);
        case MLXCAT_F16: return launch_o<__half>(kv, rope, a, st);
        case MLXCAT_BF16: return launch_o<__nv_bfloat16>(kv, rope, a, st);
    }
    return cudaErrorInvalidValue;
}

}  // namespace mlxcat
