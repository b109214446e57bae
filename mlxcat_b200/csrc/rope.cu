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
// Every input is read and every output written once.  A warp takes one token, or
// some of its heads when tokens are few, forms the angles once (a lane two pairs,
// through shared memory) and goes over the heads with the next ones' loads in
// flight.  A lane owns features d0..d0+7 and D/2 + d0..+7 of a head: the half
// layout's partners over the whole head are then in one lane, the sum of squares
// needs three shuffles (D = 128), and every access is 16 bytes.  A CTA per token
// spent most of its time on the chain position -> angles -> barrier (133 us for
// 16,396 tokens of 32 + 2 * 8 heads, bf16, normalised, interleaved), groups of four
// tokens a CTA still on the barrier (89 us), a warp a token with every lane
// choosing between q, k and v for itself 80 us; now 73 us, 5.5 TB/s, 0.84 of the
// copy rate, and the instruction rate bounds it (70 % of issue slots).  160 tokens
// of an fp32 projection: 4.5 to 4.9 us, launch-bound.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace mlxcat {

namespace {

constexpr int RA_THREADS = 256;
constexpr int RA_BATCH = 2;   // rounds of heads whose loads are in flight together
template <typename TI>
constexpr int ra_ctas() { return sizeof(TI) == 4 ? 2 : 3; }   // per SM: fp32 inputs take twice the registers

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

// two values rounded into one 32-bit word
template <typename T>
__device__ __forceinline__ uint32_t from_2f(float a, float b);
template <>
__device__ __forceinline__ uint32_t from_2f<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t from_2f<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Two fp32 values in one register pair: products and sums of both in one
// instruction (the kernel is bound by its instruction rate before it is by HBM).
__device__ __forceinline__ uint64_t two(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float lo(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float hi(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// 8 consecutive elements as they lie in memory, converted when they are used
template <typename TI>
struct Vec8 {
    static constexpr int W = sizeof(TI) / 2;   // 16-byte words
    uint4 w[W];
    __device__ __forceinline__ void load(const TI *p) {
#pragma unroll
        for (int i = 0; i < W; ++i)   // volatile: behind griddep_wait; nothing the kernel writes is read here
            asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n"
                         : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w)
                         : "l"(reinterpret_cast<const uint4 *>(p) + i));
    }
    __device__ __forceinline__ void get(uint64_t *x) const {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            x[i] = two(to_f<TI>(reinterpret_cast<const TI *>(w)[2 * i]), to_f<TI>(reinterpret_cast<const TI *>(w)[2 * i + 1]));
    }
};

// Where the partner of a feature's pair is.  A thread holds features d0..d0+7
// and D/2 + d0..+7 of a head.  OWN: next to it (interleaved layout, or no
// rotation); HALF: at the same place of the thread's other 8 (half layout, whole
// head); LANE: at the same place of another lane's first 8 (half layout, at most
// half the head, half the rotary width a multiple of 8); ANY: read again.
enum Partner { OWN, HALF, LANE, ANY };

// MIXED: a round's heads may be of more than one kind (q, k, v); else the kind is
// the round's and costs the lanes no selections.
template <typename TI, typename TO, int D, int PARTNER, bool MIXED>
__global__ void __launch_bounds__(RA_THREADS, ra_ctas<TI>())
rope_append_kernel(const PagedKV kv, const __grid_constant__ mlxcat_rope rope, const RopeAppendArgs a, int chunks, int per) {
    constexpr int LPH = D / 16, HPI = 32 / LPH;   // lanes per head, heads of a warp at a time
    __shared__ __align__(16) float cosv[RA_THREADS / 32][D / 2], sinv[RA_THREADS / 32][D / 2];
    __shared__ __align__(16) float nw[2][D];
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int nq = a.q ? a.n_heads : 0, heads = nq + 2 * kv.n_kv;
    const int j = lane % LPH, d0 = j * 8, hl0 = lane / LPH;
    const int half = a.with_rope ? rope.rotary_dim / 2 : 0;
    const bool norms = a.q_norm || a.k_norm;
    float *cw = cosv[warp], *sw = sinv[warp];
    griddep_launch_dependents();
    griddep_wait();
    if (norms) {
        for (int i = threadIdx.x; i < 2 * D; i += blockDim.x) {
            const float *w = i < D ? a.q_norm : a.k_norm;
            if (w) nw[i / D][i % D] = w[i % D];
        }
        __syncthreads();
    }
    // a unit: `per` rounds of HPI heads of one token; a warp takes every n-th unit
    const int units = a.M * chunks, nwarps = gridDim.x * (RA_THREADS / 32);
    int u = blockIdx.x * (RA_THREADS / 32) + warp;
    if (u >= units) return;
    auto fetch = [&](int m, int h0, int round, Vec8<TI> (*in)[2]) {
        const int hb = h0 + round * HPI + hl0;
#pragma unroll
        for (int b = 0; b < RA_BATCH; ++b) {
            const int hh = hb + b * HPI, kd = MIXED ? hh : hh - hl0;
            if (round + b < per && kd < heads) {
                const bool is_q = kd < nq, is_v = kd >= nq + kv.n_kv;
                const TI *p = reinterpret_cast<const TI *>(is_q ? a.q : is_v ? a.v : a.k) +
                              (int64_t)m * (int)(is_q ? a.q_stride : is_v ? a.v_stride : a.k_stride) +
                              (is_q ? hh : is_v ? hh - nq - kv.n_kv : hh - nq) * D + d0;
                in[b][0].load(p);
                in[b][1].load(p + D / 2);
            }
        }
    };
    Vec8<TI> cur[RA_BATCH][2], nxt[RA_BATCH][2];
    int m = u / chunks, h0 = (u - m * chunks) * per * HPI, mn = m, hn = h0;   // of this unit and the next
    fetch(m, h0, 0, cur);
    int row = load_id(a.trow + m), pos = load_id(a.tpos + m);
    for (; u < units; u += nwarps, m = mn, h0 = hn) {
        // the token's slot; one outside the table or the cache is not written
        int bad = 0, page = 0;
        if (row >= kv.rows) bad = PE_ROW;
        else if (pos < 0 || pos >= paged_capacity(kv)) bad = PE_POS;
        else if (row >= 0) {
            page = load_id(kv.table + (size_t)row * kv.max_pages + (pos >> kv.page_shift));
            if (page < 0 || page >= kv.n_pages) bad = PE_PAGE;
        }
        const int64_t at = bad ? -1 : (int64_t)page * kv.page_stride + (int64_t)(pos & ((1 << kv.page_shift) - 1)) * kv.token_stride;
        const bool on = row >= 0;   // else padding
        if (on && bad && lane == 0 && a.err) atomicExch(a.err, bad);
        // angles
        __syncwarp();
        for (int i = lane; i < half; i += 32) {
            const double x = (double)pos * rope.turns[i];
            float s, c;
            sincospif(2.0f * (float)(x - rint(x)), &s, &c);
            cw[i] = c * rope.mscale;
            sw[i] = s * rope.mscale;
        }
        __syncwarp();
        // what this lane's features turn by in every head (HALF: pairs d0..d0+7; OWN: d0/2..+3 and D/4 + d0/2..+3)
        float cs[8], sn[8];
        if (half && (PARTNER == HALF || PARTNER == OWN)) {
            const int p0 = PARTNER == HALF ? d0 : d0 / 2, p1 = PARTNER == HALF ? d0 + 4 : D / 4 + d0 / 2;
            *reinterpret_cast<float4 *>(cs) = *reinterpret_cast<const float4 *>(cw + p0);
            *reinterpret_cast<float4 *>(cs + 4) = *reinterpret_cast<const float4 *>(cw + p1);
            *reinterpret_cast<float4 *>(sn) = *reinterpret_cast<const float4 *>(sw + p0);
            *reinterpret_cast<float4 *>(sn + 4) = *reinterpret_cast<const float4 *>(sw + p1);
        }
        if (u + nwarps < units) {
            mn = (u + nwarps) / chunks;
            hn = (u + nwarps - mn * chunks) * per * HPI;
            row = load_id(a.trow + mn);
            pos = load_id(a.tpos + mn);
        }
#pragma unroll 1
        for (int round = 0; round < per; round += RA_BATCH) {
            if (round + RA_BATCH < per) fetch(m, h0, round + RA_BATCH, nxt);
            else if (u + nwarps < units) fetch(mn, hn, 0, nxt);
#pragma unroll
            for (int b = 0; b < RA_BATCH; ++b) {
                const int hb = h0 + (round + b) * HPI, hh = hb + hl0;
                if (!on || round + b >= per || hb >= heads) break;   // uniform: every lane shuffles
                const int kd = MIXED ? hh : hb;
                const bool in = kd < heads, is_q = kd < nq, is_v = kd >= nq + kv.n_kv;
                uint64_t x[2][4];
                cur[b][0].get(x[0]);
                cur[b][1].get(x[1]);
                const bool norm = is_q ? a.q_norm != nullptr : !is_v && a.k_norm != nullptr;
                const float *w = nw[is_q ? 0 : 1];
                float r = 1.f;
                if (norms) {
                    uint64_t s2 = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) s2 = fma2(x[i >> 2][i & 3], x[i >> 2][i & 3], s2);
                    float ss = lo(s2) + hi(s2);
#pragma unroll
                    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    if (norm) {
                        r = rsqrtf(ss * (1.0f / D) + a.eps);
                        const uint64_t r2 = two(r, r);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float4 w4 = *reinterpret_cast<const float4 *>(w + (i >> 1) * (D / 2) + d0 + (i & 1) * 4);
                            uint64_t *y = &x[i >> 1][(i & 1) * 2];
                            y[0] = mul2(mul2(y[0], r2), two(w4.x, w4.y));
                            y[1] = mul2(mul2(y[1], r2), two(w4.z, w4.w));
                        }
                    }
                }
                const bool turn = half && !is_v;
                if (PARTNER == HALF) {
                    if (turn) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint64_t c2 = two(cs[2 * i], cs[2 * i + 1]), s2 = two(sn[2 * i], sn[2 * i + 1]);
                            const uint64_t e = x[0][i], f = x[1][i], fs = mul2(f, s2);
                            x[0][i] = fma2(e, c2, two(-lo(fs), -hi(fs)));
                            x[1][i] = fma2(f, c2, mul2(e, s2));
                        }
                    }
                } else if (PARTNER == OWN) {
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const int n = half - (v * (D / 2) + d0) / 2;   // pairs of this 8 that turn
                        if (turn && n >= 4) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float e = lo(x[v][i]), f = hi(x[v][i]);
                                x[v][i] = two(e * cs[v * 4 + i] - f * sn[v * 4 + i], f * cs[v * 4 + i] + e * sn[v * 4 + i]);
                            }
                        } else if (turn && n > 0) {
#pragma unroll
                            for (int i = 0; i < 3; ++i) {
                                const float e = lo(x[v][i]), f = hi(x[v][i]);
                                if (i < n) x[v][i] = two(e * cs[v * 4 + i] - f * sn[v * 4 + i], f * cs[v * 4 + i] + e * sn[v * 4 + i]);
                            }
                        }
                    }
                } else if (PARTNER == LANE) {
                    const int hv = half >> 3, from = lane + (j < 2 * hv ? (j < hv ? hv : -hv) : 0);
                    const int p = j < hv ? d0 : d0 - half;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint64_t y = __shfl_sync(0xffffffffu, x[0][i], from);
                        if (turn && j < 2 * hv) {
                            const float2 c2 = *reinterpret_cast<const float2 *>(cw + p + 2 * i), s2 = *reinterpret_cast<const float2 *>(sw + p + 2 * i);
                            x[0][i] = fma2(y, j < hv ? two(-s2.x, -s2.y) : two(s2.x, s2.y), mul2(x[0][i], two(c2.x, c2.y)));
                        }
                    }
                } else if (turn && in) {
                    const TI *head = reinterpret_cast<const TI *>(is_q ? a.q : a.k) + (int64_t)m * (int)(is_q ? a.q_stride : a.k_stride) +
                                     (is_q ? hh : hh - nq) * D;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int d = (i >> 3) * (D / 2) + d0 + (i & 7), e = d < half ? d + half : d - half;
                        if (d >= 2 * half) continue;
                        float y = to_f<TI>(head[e]);
                        if (norm) y = y * r * w[e];
                        const int p = d < half ? d : e;
                        const uint64_t o = x[i >> 3][(i & 7) >> 1];
                        const float z = (i & 1) ? hi(o) : lo(o), v = d < half ? z * cw[p] - y * sw[p] : z * cw[p] + y * sw[p];
                        x[i >> 3][(i & 7) >> 1] = (i & 1) ? two(lo(o), v) : two(v, hi(o));
                    }
                }
                if (in && (is_q || at >= 0)) {
                    TO *to = is_q ? reinterpret_cast<TO *>(a.q_out) + ((int64_t)m * a.n_heads + hh) * D + d0
                                  : reinterpret_cast<TO *>(is_v ? kv.v : kv.k) + at + (int64_t)(is_v ? hh - nq - kv.n_kv : hh - nq) * kv.head_stride + d0;
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        uint4 out;
                        out.x = from_2f<TO>(lo(x[v][0]), hi(x[v][0]));
                        out.y = from_2f<TO>(lo(x[v][1]), hi(x[v][1]));
                        out.z = from_2f<TO>(lo(x[v][2]), hi(x[v][2]));
                        out.w = from_2f<TO>(lo(x[v][3]), hi(x[v][3]));
                        *reinterpret_cast<uint4 *>(to + v * (D / 2)) = out;
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < RA_BATCH; ++b) { cur[b][0] = nxt[b][0]; cur[b][1] = nxt[b][1]; }
        }
    }
}

template <typename TI, typename TO, int D, int PARTNER>
cudaError_t launch_t(const PagedKV &kv, const mlxcat_rope &rope, const RopeAppendArgs &a, cudaStream_t st) {
    constexpr int HPI = 32 / (D / 16), WARPS = RA_THREADS / 32;
    const int rounds = ((a.q ? a.n_heads : 0) + 2 * kv.n_kv + HPI - 1) / HPI;
    const int64_t wave = (int64_t)ra_ctas<TI>() * a.sm_count * WARPS;
    // few tokens: their heads are spread over the warps of a wave; many: a warp
    // takes a token's heads one after the other and forms its angles once
    const int spread = (int)std::max<int64_t>(1, std::min<int64_t>(rounds, wave / a.M));
    const int per = (rounds + spread - 1) / spread, chunks = (rounds + per - 1) / per;
    const int64_t units = (int64_t)a.M * chunks;
    if (units > 0x3fffffff) return cudaErrorInvalidValue;
    const unsigned grid = (unsigned)std::min<int64_t>((units + WARPS - 1) / WARPS, wave / WARPS);
    if (((a.q ? a.n_heads : 0) % HPI) == 0 && kv.n_kv % HPI == 0)
        return launch_pdl(rope_append_kernel<TI, TO, D, PARTNER, false>, dim3(grid), dim3(RA_THREADS), 0, st, kv, rope, a, chunks, per);
    return launch_pdl(rope_append_kernel<TI, TO, D, PARTNER, true>, dim3(grid), dim3(RA_THREADS), 0, st, kv, rope, a, chunks, per);
}

template <typename TI, typename TO, int D>
cudaError_t launch_p(const PagedKV &kv, const mlxcat_rope &rope, const RopeAppendArgs &a, cudaStream_t st) {
    if (!a.with_rope || rope.layout == MLXCAT_ROPE_INTERLEAVED) return launch_t<TI, TO, D, OWN>(kv, rope, a, st);
    if (rope.rotary_dim == D) return launch_t<TI, TO, D, HALF>(kv, rope, a, st);
    if (rope.rotary_dim % 16 || rope.rotary_dim > D / 2) return launch_t<TI, TO, D, ANY>(kv, rope, a, st);
    return launch_t<TI, TO, D, LANE>(kv, rope, a, st);
}

template <typename TI, typename TO>
cudaError_t launch_d(const PagedKV &kv, const mlxcat_rope &rope, const RopeAppendArgs &a, cudaStream_t st) {
    return kv.D == 128 ? launch_p<TI, TO, 128>(kv, rope, a, st) : launch_p<TI, TO, 64>(kv, rope, a, st);
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
