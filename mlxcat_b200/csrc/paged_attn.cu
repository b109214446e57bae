// paged_attn.cu -- attention of single tokens and verify groups over a paged
// cache:  out[m, h] = sum_p softmax_p(scale q[m,h].k_p) v_p,  p <= tpos[m].
//
// Bound by HBM: every K and V byte of a row is read once and meets only the
// qg * G query rows of its KV head, far below the ridge.  So the kernel is a
// stream with as little between the loads as possible:
//
// * A warp owns 16 keys at a time and its own ring of cp.async stages (no CTA
//   barrier in the loop).  Pages are looked up 32 tiles at a time, a lane each.
// * The products are transposed: S^T = K Q^T with the 16 keys as the M of
//   mma.m16n8k16 and 8 query rows as its N, then O^T = V^T P^T.  A group of 4
//   or 8 query rows fills the N = 8 tile (as M it would pad to 16), and the
//   accumulator of S^T, packed to 16 bits and turned by movmatrix, is the B
//   operand of the second product.  The row sums come from the same packed P,
//   by one more product with a matrix of ones, so numerator and denominator
//   round alike.
// * P = 2^(z - m), z in log2 units; the reference m moves only when a score is
//   more than 8 above it (P <= 256 fits fp16), so most tiles have no
//   cross-lane maximum and no rescaling.
// * Rows differ in length and only the device knows it: the units (64 keys) of
//   all (group, KV head, query tile) items are laid end to end and every CTA
//   takes an equal stretch.  An item inside one CTA is finished there; the
//   others leave (O, max, sum) partials, which attn_join merges in order, so
//   results do not depend on timing.
//
// Two CTAs of four warps an SM keep 128 KB of loads in flight; with two or one
// warp a CTA (four or six CTAs) 64 rows of up to 16k keys took 395 and 308 us
// where two of four took 298.  Measured on B200s: those 64 rows (64 query heads, 8
// KV heads of 128, bf16) 303 to 307 us, 6.2 TB/s, 0.95 of the copy rate; 32 x 5 verify
// tokens over 4.2k keys 106 to 110 us, 5.0 to 5.2 TB/s.  What is left there is the
// start (the lengths, the page ids and the first keys are one chain of loads, 3 us)
// and the join.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"
#include "tc.cuh"

namespace mlxcat {

namespace {

constexpr int PW = 4;              // warps per CTA
constexpr int PT = PW * 32;
constexpr int TK = 16;             // keys per warp tile
constexpr int UNIT = PW * TK;      // keys per unit
constexpr int ST = 3;              // ring stages per warp
constexpr int CTAS_PER_SM = 2;
// An item costs a CTA about as much to begin and end (queries, page lookups, first
// loads, merge: 5,500 cycles) as three units of keys: its stretch has that many
// units without keys in front, so that CTAs of many short items are not the last.
constexpr int LEAD = 3;
constexpr int ONE_CLUSTER = 8, CLUSTER_UNITS = 8;   // CTAs of a small call's cluster, units each at most

template <typename T>
struct Half2;
template <>
struct Half2<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2 *>(&x)); }
    static constexpr uint32_t ones = 0x3C003C00u;
    static __device__ __forceinline__ void mma(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <>
struct Half2<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t x) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&x)); }
    static constexpr uint32_t ones = 0x3F803F80u;
    static __device__ __forceinline__ void mma(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

__device__ __forceinline__ void ldm4(uint32_t *d, uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t *d, uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void cpa16(uint32_t s, const void *g, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(s), "l"(g), "r"(bytes) : "memory");
}

// What a group of tokens sees: its row and one past its last key.
struct Group {
    int row, kend;
};
// the same, clamped to what the table holds; the flag where it was not
__device__ __forceinline__ Group checked(const PagedKV &kv, const PagedQuery &a, Group x) {
    const int cap = paged_capacity(kv);
    if (x.row >= kv.rows || x.kend > cap) {
        if (a.err) atomicExch(a.err, x.row >= kv.rows ? PE_ROW : PE_POS);
        x.kend = x.row >= kv.rows ? 0 : cap;
    }
    if (x.row < 0) x.kend = 0;
    return x;
}
__device__ __forceinline__ Group group_alone(const PagedKV &kv, const PagedQuery &a, int grp) {
    const int t0 = grp * a.qg, n = min(a.qg, a.M - t0);
    Group x = {-1, 0};
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
        const int r = load_id(a.trow + t0 + j), p = load_id(a.tpos + t0 + j);
        if (r >= 0) {
            x.row = max(x.row, r);
            x.kend = max(x.kend, p == 0x7fffffff ? p : p + 1);
        }
    }
    return checked(kv, a, x);
}

__device__ __forceinline__ int64_t cta_begin(int c, int64_t U, int C) { return (int64_t)c * U / C; }

// What a partial with maximum m and sum l weighs against the maximum mx of all.
// A partial that saw nothing (m = -inf, l = 0) weighs nothing; one whose scores
// were all NaN keeps its NaN sum.
__device__ __forceinline__ float weight_of(float m, float l, float mx) {
    return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : tc::ex2_approx(m - mx);
}

// Shared memory: the warps' rings, the item's query rows, their limits.  The
// merge of the warps has its own memory where two CTAs of an SM have room for it
// (EARLY: the next piece's loads then run during the merge), else the rings'.
template <int D, int NT>
struct PagedShape {
    static constexpr int STAGE = 2 * TK * D * 2;            // K and V of one tile, bytes
    static constexpr int RING = PW * ST * STAGE;
    static constexpr int QR = NT * 8;                       // query rows of an item
    static constexpr int MT = D / 16, MTW = MT / PW;        // m tiles of O^T, and those a warp finishes
    static constexpr int FRAGS = PW * (PW - 1) * MTW * NT * 512;   // what the warps hand to one another
    static constexpr int MERGE = FRAGS + PW * QR * 8;
    static constexpr int TAIL = QR * D * 2 + QR * 4;
    // the query operands stay in registers for two n8 tiles at most
    static constexpr bool QREG = NT <= 2 || D == 64;
    static constexpr bool EARLY = QREG && RING + MERGE + TAIL + 2304 <= (228 * 1024) / CTAS_PER_SM - 1024;
    static constexpr int BODY = EARLY ? RING + MERGE : RING > MERGE ? RING : MERGE;
    static constexpr int MERGE_AT = EARLY ? RING : 0;
    static constexpr int SMEM = BODY + TAIL;
};
constexpr int NOBODY = 0x7fffffff;   // key limit of query rows that are padding or behind the group
// Groups whose (row, last key) a CTA keeps; beyond, it reads them again from the
// descriptors.  Rows of 1,024 keys (32 / 8 heads of 128): 256 rows 178 us, 257 180,
// 512 340, 2,048 1,340; groups of 5 tokens: 256 rows 224 us, 257 223, 512 398.
constexpr int MAX_GROUPS = 256;

// 8 features of a query row on their way through partials.
struct Joined {
    float mx = -INFINITY, l = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
};

// Merge an item's pieces (and, after a shared prefix, the prefix's splits) by a
// whole CTA: a thread takes 8 features of a query row and every P-th piece, in
// order (P > 1 when there are more than one round of loads); P such threads then add up through shared memory (10 floats a thread).
template <typename T, int D>
__device__ __forceinline__ void join_item(const PagedKV &kv, const PagedQuery &a, int QR, size_t item,
                                          const float *o_part, const float *ml_part, int2 mt, const PrefixPartials &pre,
                                          float *sm) {
    const int Hq = a.n_heads, G = Hq / kv.n_kv;
    const int qts = (a.qg * G + QR - 1) / QR, per_group = kv.n_kv * qts;
    const int grp = (int)(item / per_group), x = (int)(item % per_group), h = x / qts, qt = x - h * qts;
    if (mt.y < 0 && pre.splits == 0) return;   // written already
    const int t0 = grp * a.qg, ntok = min(a.qg, a.M - t0);
    const int nq = min(QR, ntok * G - qt * QR), W = nq * (D / 8);
    const int n_own = mt.y >= 0 ? mt.y - mt.x + 1 : 0, n = n_own + pre.splits;
    if (W <= 0) return;
    constexpr int PB = 8;   // pieces whose loads are in flight together
    auto gather = [&](int w, int first, int step, Joined &j) {
        const int r = w / (D / 8), d = (w % (D / 8)) * 8, rr = qt * QR + r;
        for (int p0 = first; p0 < n; p0 += PB * step) {
            float2 ml[PB];
            float4 va[PB], vb[PB];
#pragma unroll
            for (int k = 0; k < PB; ++k) {
                ml[k] = make_float2(-INFINITY, 0.f);
                va[k] = vb[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                const int p = p0 + k * step;
                if (p < n) {
                    const float *o, *q;
                    if (p < n_own) {
                        const size_t at = (item + mt.x + p) * QR + r;
                        o = o_part + at * D + d;
                        q = ml_part + at * 2;
                    } else {   // [split][KV head][8 features][row][8]
                        const size_t rows = (size_t)a.M * G, sh = (size_t)(p - n_own) * kv.n_kv + h, row = (size_t)t0 * G + rr;
                        o = pre.o + ((sh * (D / 8) + d / 8) * rows + row) * 8;
                        q = pre.ml + (sh * rows + row) * 2;
                    }
                    ml[k] = *reinterpret_cast<const float2 *>(q);
                    va[k] = *reinterpret_cast<const float4 *>(o);
                    vb[k] = *reinterpret_cast<const float4 *>(o + 4);
                }
            }
            float mb = j.mx;
#pragma unroll
            for (int k = 0; k < PB; ++k) mb = fmaxf(mb, ml[k].x);
            if (j.mx != -INFINITY && j.mx != mb) {
                const float f = tc::ex2_approx(j.mx - mb);
                j.l *= f;
#pragma unroll
                for (int i = 0; i < 8; ++i) j.acc[i] *= f;
            }
            j.mx = mb;
#pragma unroll
            for (int k = 0; k < PB; ++k) {
                const float f = weight_of(ml[k].x, ml[k].y, mb);
                j.l += f * ml[k].y;
                j.acc[0] += f * va[k].x; j.acc[1] += f * va[k].y; j.acc[2] += f * va[k].z; j.acc[3] += f * va[k].w;
                j.acc[4] += f * vb[k].x; j.acc[5] += f * vb[k].y; j.acc[6] += f * vb[k].z; j.acc[7] += f * vb[k].w;
            }
        }
    };
    // asked before the pieces are gathered, so that the load is not one more in the chain
    auto padding = [&](int w) { return load_id(a.trow + t0 + (qt * QR + w / (D / 8)) / G) < 0; };
    auto write = [&](int w, const Joined &j) {
        const int r = w / (D / 8), d = (w % (D / 8)) * 8, rr = qt * QR + r, m = t0 + rr / G;
        const float inv = j.l != 0.f ? 1.f / j.l : 0.f;
        uint4 y;
        y.x = Half2<T>::pack(j.acc[0] * inv, j.acc[1] * inv);
        y.y = Half2<T>::pack(j.acc[2] * inv, j.acc[3] * inv);
        y.z = Half2<T>::pack(j.acc[4] * inv, j.acc[5] * inv);
        y.w = Half2<T>::pack(j.acc[6] * inv, j.acc[7] * inv);
        *reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + ((size_t)m * Hq + h * G + rr % G) * D + d) = y;
    };
    const int P = min((int)blockDim.x / W, (n + PB - 1) / PB);
    if (P <= 1) {
        for (int w = threadIdx.x; w < W; w += blockDim.x) {
            Joined j;
            const bool pad = padding(w);
            gather(w, 0, 1, j);
            if (!pad) write(w, j);
        }
        return;
    }
    const int g = threadIdx.x / W, w = threadIdx.x % W;
    Joined j;
    const bool pad = g || padding(w);
    if (g < P) gather(w, g, P, j);
    float *mine = sm + threadIdx.x;
    const int bs = blockDim.x;
    mine[0] = j.mx;
    mine[bs] = j.l;
#pragma unroll
    for (int i = 0; i < 8; ++i) mine[(2 + i) * bs] = j.acc[i];
    __syncthreads();
    if (!pad) {
        float mx = j.mx;
        for (int p = 1; p < P; ++p) mx = fmaxf(mx, sm[p * W + w]);
        Joined t;
        for (int p = 0; p < P; ++p) {
            const float *o = sm + p * W + w;
            const float f = weight_of(o[0], o[bs], mx);
            t.l += f * o[bs];
#pragma unroll
            for (int i = 0; i < 8; ++i) t.acc[i] += f * o[(2 + i) * bs];
        }
        write(w, t);
    }
    __syncthreads();   // before the next item's
}

template <typename T, int D>
__global__ void __launch_bounds__(256)
attn_join(const PagedKV kv, const PagedQuery a, int QR, const float *__restrict__ o_part,
          const float *__restrict__ ml_part, const int2 *__restrict__ meta, const PrefixPartials pre) {
    __shared__ float sm[10 * 256];
    griddep_launch_dependents();
    griddep_wait();
    if (pre.splits && blockIdx.x == 0 && threadIdx.x == 0) *pre.ready = 0;   // for a replay of this call
    join_item<T, D>(kv, a, QR, blockIdx.x, o_part, ml_part, meta[blockIdx.x], pre, sm);
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(PT, CTAS_PER_SM)
paged_attn_kernel(const PagedKV kv, const PagedQuery a, int key_begin, int force_partial, float *o_part, float *ml_part,
                  int2 *meta, const PrefixPartials pre, int one_cluster, int items) {
    using S = PagedShape<D, NT>;
    constexpr int CH = D / 8;            // 16-byte chunks per key
    constexpr int RPI = 32 / CH;         // keys per load instruction of a warp
    // Up to two n8 tiles the kernel waits for HBM, not for the tensor cores: P goes in
    // as two 16-bit parts and keeps 21 (bf16: 16) bits, so the result's own rounding is
    // the only one that shows (64 single tokens over up to 16k keys: 298 us either way).
    // With three tiles it cost 105 -> 117 us at 32 x 5 tokens over 4.2k keys.
    constexpr bool TWO = NT <= 2;
    extern __shared__ __align__(128) unsigned char psm[];
    unsigned char *qsm = psm + S::BODY;                                       // [QR][D], chunks swizzled
    int *lim_s = reinterpret_cast<int *>(qsm + S::QR * D * 2);                // [QR]
    __shared__ int64_t wsum[PW];
    __shared__ int64_t start_s[2];       // group of the first unit, units before it
    __shared__ Group info[MAX_GROUPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const int Hq = a.n_heads, Hkv = kv.n_kv, G = Hq / Hkv;
    const int groups = (a.M + a.qg - 1) / a.qg;
    const int qts = (a.qg * G + S::QR - 1) / S::QR;
    const int per_group = Hkv * qts;     // items of a group: (query tile, KV head)
    const uint32_t inv_g = (uint32_t)((0x100000000ull + G - 1) / G);   // row / G by one product: row < 2^26
    auto div_g = [&](int x) { return G == 1 ? x : (int)__umulhi((uint32_t)x, inv_g); };
    // units of an item of the group, the leading ones among them; 0 without keys
    auto units_of = [&](const Group &x) { return x.kend > key_begin ? (x.kend - key_begin + UNIT - 1) / UNIT + LEAD : 0; };

    // Behind a prefix pass this kernel needs nothing of it: it starts on the SMs the
    // pass leaves free (which itself lets it start only once all before the pass is
    // done) and waits at its end, so that the join after it waits for both.  That what
    // was written before the pass is visible here does not follow from the early start:
    // the pass releases its sign once it has waited for those writes, and this kernel
    // acquires it.  A CTA that does not find the sign yet waits for the pass (all of
    // them waiting at once: 64 tokens over an 8k document 42 -> 65 us).
    griddep_launch_dependents();
    bool ordered = false;
    if (force_partial) {
        if (threadIdx.x == 0) ordered = tc::ld_acquire_gpu(pre.ready) == pre.token;
        ordered = __syncthreads_or(ordered);
    }
    if (!ordered) griddep_wait();

    // ---- where this CTA's stretch of units starts: thread x sums the groups of
    // its chunk, a scan gives the total and the chunk that holds the start
    const int per = (groups + PT - 1) / PT;
    const bool kept = groups <= MAX_GROUPS;
    int64_t mine = 0;
    if (kept && a.qg > 1) {
        // a thread per token, so that all loads are one round trip; a group's row and
        // last key are maxima
        for (int i = threadIdx.x; i < groups; i += PT) info[i] = {-1, 0};
        __syncthreads();
#pragma unroll 2
        for (int m = threadIdx.x; m < a.M; m += PT) {
            const int r = load_id(a.trow + m), p = load_id(a.tpos + m), i = m / a.qg;
            if (r >= 0) {
                atomicMax(&info[i].row, r);
                atomicMax(&info[i].kend, p == 0x7fffffff ? p : p + 1);
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < groups; i += PT) info[i] = checked(kv, a, info[i]);
        __syncthreads();
    }
    {
        const int g0 = threadIdx.x * per, g1 = min(groups, g0 + per);
        for (int i = g0; i < g1; ++i) {
            const bool known = kept && a.qg > 1;
            const Group x = known ? info[i] : group_alone(kv, a, i);
            if (kept && !known) info[i] = x;
            mine += units_of(x);
        }
    }
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    auto group = [&](int i) { return kept ? info[i] : group_alone(kv, a, i); };
    int64_t before = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < PW; ++w) {
        if (w < warp) before += wsum[w];
        total += wsum[w];
    }
    const int64_t U = total * per_group;
    const int C = (int)min((int64_t)gridDim.x, U);   // CTAs that work
    const int64_t u0 = blockIdx.x < C ? cta_begin(blockIdx.x, U, C) : 0;
    const int64_t u1 = blockIdx.x < C ? cta_begin(blockIdx.x + 1, U, C) : 0;
    if (u1 > u0 && before * per_group <= u0 && u0 < (before + mine) * per_group) {
        int64_t acc = before * per_group;
        int i = threadIdx.x * per;
        for (;; ++i) {
            const int64_t n = (int64_t)units_of(group(i)) * per_group;
            if (u0 < acc + n) break;
            acc += n;
        }
        start_s[0] = i;
        start_s[1] = acc;
    }
    __syncthreads();

    // ---- groups without keys here: nothing else writes their outputs
    for (int i = blockIdx.x * PW + warp; i < groups; i += gridDim.x * PW) {
        if (units_of(group(i))) continue;
        for (int x = lane; x < per_group; x += 32) meta[(size_t)i * per_group + x] = make_int2(0, -1);
        if (force_partial) continue;
        const int t0 = i * a.qg, n = min(a.qg, a.M - t0);
        for (int j = 0; j < n; ++j) {
            if (load_id(a.trow + t0 + j) < 0) continue;   // padding stays as it was
            uint4 *dst = reinterpret_cast<uint4 *>(reinterpret_cast<T *>(a.out) + (size_t)(t0 + j) * Hq * D);
            for (int x = lane; x < Hq * D / 8; x += 32) dst[x] = make_uint4(0, 0, 0, 0);
        }
    }
    const bool work = u1 > u0;
    int grp = work ? (int)start_s[0] : 0;
    int64_t ubase = work ? start_s[1] : 0;   // units before this group
    Group gi = group(grp);
    int gu = units_of(gi);               // units per item
    unsigned char *ring = psm + warp * (ST * S::STAGE);
    const uint32_t ring_a = tc::smem_u32(ring), qsm_a = tc::smem_u32(qsm);
    const int ch = lane % CH, r0 = lane / CH;

    // A piece: this CTA's part of an item.
    struct Piece {
        int64_t ib;             // the item's first unit
        size_t item;
        const T *kb, *vb;
        const int32_t *table;
        int gu, h, qt, t0, nq, kend, ua, steps, kfirst;
        bool whole;
    };
    int64_t u = u0;
    auto next_piece = [&](Piece &p) -> bool {
        while (u < u1) {
            while (u >= ubase + (int64_t)gu * per_group) {
                ubase += (int64_t)gu * per_group;
                gi = group(++grp);
                gu = units_of(gi);
            }
            const int x = (int)((u - ubase) / gu);                 // item of the group
            p.ib = ubase + (int64_t)x * gu;
            const int va = (int)(u - p.ib), vend = (int)min((int64_t)gu, u1 - p.ib);
            u = p.ib + vend;
            p.ua = max(va - LEAD, 0);
            p.steps = vend - LEAD - p.ua;                          // units of keys
            if (p.steps <= 0) continue;                            // leading units only
            p.whole = p.ua == 0 && vend == gu;
            p.gu = gu;
            p.h = x / qts;
            p.qt = x - p.h * qts;
            p.t0 = grp * a.qg;
            p.nq = min(S::QR, min(a.qg, a.M - p.t0) * G - p.qt * S::QR);   // may be <= 0 in a last, short group
            p.item = (size_t)grp * per_group + x;
            p.kend = gi.kend;
            p.kfirst = key_begin + p.ua * UNIT + warp * TK;        // key 0 of step 0 (fits: below the table's capacity + UNIT)
            p.kb = reinterpret_cast<const T *>(kv.k) + (int64_t)p.h * kv.head_stride;
            p.vb = reinterpret_cast<const T *>(kv.v) + (int64_t)p.h * kv.head_stride;
            p.table = kv.table + (size_t)gi.row * kv.max_pages;
            return true;
        }
        return false;
    };
    const int pmask = (1 << kv.page_shift) - 1;
    int pid[2] = {-1, -1};       // lane l: pages of the two 8-key halves of step (32 batch + l)
    auto stage = [&](const Piece &p, int s) {
        if ((s & 31) == 0) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int64_t key = (int64_t)p.kfirst + (int64_t)(s + lane) * UNIT + 8 * e;
                int id = -1;
                if (s + lane < p.steps && key < p.kend) {
                    id = load_id(p.table + (key >> kv.page_shift));
                    if (id < 0 || id >= kv.n_pages) {
                        id = -1;
                        if (a.err) atomicExch(a.err, PE_PAGE);
                    }
                }
                pid[e] = id;
            }
        }
        const int p0 = __shfl_sync(0xffffffffu, pid[0], s & 31), p1 = __shfl_sync(0xffffffffu, pid[1], s & 31);
        const uint32_t dst = ring_a + (uint32_t)(s % ST) * S::STAGE;
        const int key0 = p.kfirst + s * UNIT;
#pragma unroll
        for (int i = 0; i < TK / RPI; ++i) {
            const int r = r0 + i * RPI, key = key0 + r;
            const int id = r < 8 ? p0 : p1;
            const bool ok = key < p.kend && id >= 0;
            const int64_t off = ok ? (int64_t)id * kv.page_stride + (int64_t)(key & pmask) * kv.token_stride + ch * 8 : 0;
            const uint32_t so = dst + (uint32_t)(r * D * 2 + ((ch ^ (r & 7)) << 4));
            cpa16(so, p.kb + off, ok ? 16 : 0);
            cpa16(so + TK * D * 2, p.vb + off, ok ? 16 : 0);
        }
    };
    // the piece's query rows and key limits into shared memory, its first tiles into the ring
    auto begin = [&](const Piece &p) {
        for (int w = threadIdx.x; w < S::QR * CH; w += PT) {
            const int r = w / CH, c = w % CH, rr = p.qt * S::QR + r, j = div_g(rr);
            const bool ok = r < p.nq;
            const T *src = reinterpret_cast<const T *>(a.q) + ((size_t)(p.t0 + (ok ? j : 0)) * Hq + p.h * G + (ok ? rr - j * G : 0)) * D + c * 8;
            cpa16(qsm_a + (uint32_t)(r * D * 2 + ((c ^ (r & 7)) << 4)), src, ok ? 16 : 0);
        }
        if (threadIdx.x < S::QR) {
            const int r = threadIdx.x, m = p.t0 + div_g(p.qt * S::QR + r);
            // rows nobody reads see everything: they need no mask (no position is beyond NOBODY - 1:
            // the table ends before it)
            lim_s[r] = r < p.nq && load_id(a.trow + m) >= 0 ? min(load_id(a.tpos + m), NOBODY - 1) : NOBODY;
        }
#pragma unroll
        for (int s = 0; s < ST - 1; ++s) {
            if (s < p.steps) stage(p, s);
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        }
    };

    Piece pc, pn;
    bool have = next_piece(pc);
    if (have) begin(pc);
    while (have) {
        const int qt = pc.qt, h = pc.h, t0 = pc.t0, nq = pc.nq;
        float o[D / 16][NT][4], ls[NT][4], mr[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            mr[nt][0] = mr[nt][1] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) ls[nt][i] = 0.f;
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[mt][nt][i] = 0.f;
        }
        asm volatile("cp.async.wait_group %0;\n" ::"n"(ST - 2) : "memory");   // the queries came with the first stage
        __syncthreads();
        // query rows as B operands, key limits of this lane's columns
        uint32_t qf[NT][D / 16][2];
        int lim[NT][2];
        int lim_min = NOBODY;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * 8 + (lane & 7);
#pragma unroll
            for (int ks = 0; ks < D / 16; ks += 2)
                if (S::QREG) ldm4(&qf[nt][ks][0], qsm_a + (uint32_t)(r * D * 2 + (((ks * 2 + (lane >> 3)) ^ (r & 7)) << 4)));
            lim[nt][0] = lim_s[nt * 8 + 2 * t];
            lim[nt][1] = lim_s[nt * 8 + 2 * t + 1];
            lim_min = min(lim_min, min(lim[nt][0], lim[nt][1]));
        }
        lim_min = __reduce_min_sync(0xffffffffu, lim_min);
        if (S::EARLY) __syncthreads();   // the next piece's may come in
        for (int s = 0; s < pc.steps; ++s) {
            __syncwarp();            // every lane has read the stage that is filled now
            if (s + ST - 1 < pc.steps) stage(pc, s + ST - 1);
            asm volatile("cp.async.commit_group;\n" ::: "memory");
            asm volatile("cp.async.wait_group %0;\n" ::"n"(ST - 1) : "memory");
            __syncwarp();
            const int key0 = pc.kfirst + s * UNIT;
            if (key0 >= pc.kend) continue;   // no key of this tile (a last unit)
            const uint32_t ka = ring_a + (uint32_t)(s % ST) * S::STAGE, va = ka + TK * D * 2;
            float sc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
            {
                const int r = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
                for (int ks = 0; ks < D / 16; ks += 2) {
                    uint32_t f[2][4];
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        ldm4(f[e], ka + (uint32_t)(r * D * 2 + ((((ks + e) * 2 + (lane >> 4)) ^ (r & 7)) << 4)));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        uint32_t q[4];
                        if (S::QREG) {
                            q[0] = qf[nt][ks][0]; q[1] = qf[nt][ks][1]; q[2] = qf[nt][ks + 1][0]; q[3] = qf[nt][ks + 1][1];
                        } else {
                            const int qr = nt * 8 + (lane & 7);
                            ldm4(q, qsm_a + (uint32_t)(qr * D * 2 + (((ks * 2 + (lane >> 3)) ^ (qr & 7)) << 4)));
                        }
                        Half2<T>::mma(sc[nt], f[0], q[0], q[1]);
                        Half2<T>::mma(sc[nt], f[1], q[2], q[3]);
                    }
                }
            }
            if (key0 + TK - 1 > lim_min || key0 + TK > pc.kend) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = key0 + g + (i >> 1) * 8;
                        if (key > lim[nt][i & 1] || key >= pc.kend) sc[nt][i] = -INFINITY;
                    }
            }
            bool raise = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sc[nt][i] *= a.scale_log2;
                    raise |= sc[nt][i] > mr[nt][i & 1] + 8.f;
                }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(sc[nt][e], sc[nt][2 + e]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float mn = fmaxf(mr[nt][e], mx);
                        const float al = mr[nt][e] == -INFINITY ? 0.f : tc::ex2_approx(mr[nt][e] - mn);
                        mr[nt][e] = mn;
                        ls[nt][e] *= al;
#pragma unroll
                        for (int mt = 0; mt < D / 16; ++mt) {
                            o[mt][nt][e] *= al;
                            o[mt][nt][2 + e] *= al;
                        }
                    }
            }
            uint32_t pb[NT][2], pl[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float n0 = mr[nt][0] == -INFINITY ? 0.f : mr[nt][0], n1 = mr[nt][1] == -INFINITY ? 0.f : mr[nt][1];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float p0 = tc::ex2_approx(sc[nt][2 * e] - n0), p1 = tc::ex2_approx(sc[nt][2 * e + 1] - n1);
                    const uint32_t hi = Half2<T>::pack(p0, p1);
                    pb[nt][e] = turn8x8(hi);
                    if (TWO) {   // what the rounding left out
                        const float2 h = Half2<T>::unpack(hi);
                        pl[nt][e] = turn8x8(Half2<T>::pack(p0 - h.x, p1 - h.y));
                    }
                }
            }
            const uint32_t one[4] = {Half2<T>::ones, Half2<T>::ones, Half2<T>::ones, Half2<T>::ones};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                Half2<T>::mma(ls[nt], one, pb[nt][0], pb[nt][1]);
                if (TWO) Half2<T>::mma(ls[nt], one, pl[nt][0], pl[nt][1]);
            }
            {
                const int r = (lane & 7) + (lane >> 4) * 8;
#pragma unroll
                for (int mt = 0; mt < D / 16; ++mt) {
                    uint32_t f[4];
                    ldm4t(f, va + (uint32_t)(r * D * 2 + (((mt * 2 + ((lane >> 3) & 1)) ^ (r & 7)) << 4)));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        Half2<T>::mma(o[mt][nt], f, pb[nt][0], pb[nt][1]);
                        if (TWO) Half2<T>::mma(o[mt][nt], f, pl[nt][0], pl[nt][1]);
                    }
                }
            }
        }

        // ---- merge the warps' partials: every warp finishes MTW m tiles of O^T and
        // gets the others' accumulator fragments of them ([from][to][m tile][nt][lane])
        const bool more = next_piece(pn);
        if (S::EARLY) {
            __syncwarp();   // every lane is through with the ring
            if (more) begin(pn);
        } else {
            asm volatile("cp.async.wait_group 0;\n" ::: "memory");
            __syncthreads();
        }
        float4 *of = reinterpret_cast<float4 *>(psm + S::MERGE_AT);
        float2 *mls = reinterpret_cast<float2 *>(psm + S::MERGE_AT + S::FRAGS);   // [warp][QR] (max, sum)
        auto frag = [&](int src, int mt, int nt) {
            const int to = mt / S::MTW;
            return (((src * (PW - 1) + to - (to > src)) * S::MTW + mt % S::MTW) * NT + nt) * 32 + lane;
        };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int mt = 0; mt < S::MT; ++mt)
                if (mt / S::MTW != warp) of[frag(warp, mt, nt)] = make_float4(o[mt][nt][0], o[mt][nt][1], o[mt][nt][2], o[mt][nt][3]);
            if (g == 0) {
                mls[warp * S::QR + nt * 8 + 2 * t] = make_float2(mr[nt][0], ls[nt][0]);
                mls[warp * S::QR + nt * 8 + 2 * t + 1] = make_float2(mr[nt][1], ls[nt][1]);
            }
        }
        __syncthreads();
        const bool direct = pc.whole && !force_partial;
        // slots in order of (item, CTA): unique, since a piece starts a new item or a new CTA
        const size_t slot = pc.item + blockIdx.x;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float f[2][PW], l[2], mx[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float2 ml[PW];
                mx[e] = -INFINITY;
                l[e] = 0.f;
#pragma unroll
                for (int i = 0; i < PW; ++i) {
                    ml[i] = mls[i * S::QR + nt * 8 + 2 * t + e];
                    mx[e] = fmaxf(mx[e], ml[i].x);
                }
#pragma unroll
                for (int i = 0; i < PW; ++i) {
                    f[e][i] = weight_of(ml[i].x, ml[i].y, mx[e]);
                    l[e] += f[e][i] * ml[i].y;
                }
            }
            const int ra = nt * 8 + 2 * t;                       // this lane's two query rows
            if (!direct && warp == 0 && g == 0) {
                if (ra < nq) *reinterpret_cast<float2 *>(ml_part + (slot * S::QR + ra) * 2) = make_float2(mx[0], l[0]);
                if (ra + 1 < nq) *reinterpret_cast<float2 *>(ml_part + (slot * S::QR + ra + 1) * 2) = make_float2(mx[1], l[1]);
            }
            const float inv0 = l[0] != 0.f ? 1.f / l[0] : 0.f, inv1 = l[1] != 0.f ? 1.f / l[1] : 0.f;
            // 16-bit results go out as pairs of features: even g the first row's, odd g the second's
            const int rw = ra + (g & 1), rr = qt * S::QR + rw, j = div_g(rr), m = t0 + j;
            // (without EARLY the limits in shared memory are still this piece's)
            const int own = !S::EARLY ? lim_s[rw] : (g & 1) ? lim[nt][1] : lim[nt][0];
            const bool write = rw < nq && (!direct || own != NOBODY);
            T *dst = reinterpret_cast<T *>(a.out) + ((size_t)m * Hq + h * G + rr - j * G) * D + (g & ~1);
#pragma unroll
            for (int mt = 0; mt < S::MT; ++mt) {
                if (mt / S::MTW != warp) continue;
                float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < PW; ++i) {
                    const float4 z = i == warp ? make_float4(o[mt][nt][0], o[mt][nt][1], o[mt][nt][2], o[mt][nt][3])
                                               : of[frag(i, mt, nt)];
                    y[0] += f[0][i] * z.x; y[1] += f[1][i] * z.y; y[2] += f[0][i] * z.z; y[3] += f[1][i] * z.w;
                }
                if (direct) {
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        const float v0 = y[2 * hh] * inv0, v1 = y[2 * hh + 1] * inv1;
                        const float z = __shfl_xor_sync(0xffffffffu, (g & 1) ? v0 : v1, 4);
                        if (write) *reinterpret_cast<uint32_t *>(dst + mt * 16 + hh * 8) = (g & 1) ? Half2<T>::pack(z, v1) : Half2<T>::pack(v0, z);
                    }
                } else {
                    float *dp = o_part + (slot * S::QR + ra) * D + mt * 16 + g;
                    if (ra < nq) { dp[0] = y[0]; dp[8] = y[2]; }
                    if (ra + 1 < nq) { dp[D] = y[1]; dp[D + 8] = y[3]; }
                }
            }
        }
        // the CTA that holds an item's first keys says where its pieces are
        if (pc.ua == 0 && threadIdx.x == 0) {
            const int last = (int)(((pc.ib + pc.gu) * C - 1) / U);
            meta[pc.item] = direct ? make_int2(0, -2) : make_int2(blockIdx.x, last);
        }
        __syncthreads();   // the merge's memory is used again
        if (!S::EARLY && more) begin(pn);
        pc = pn;
        have = more;
    }
    if (force_partial) griddep_wait();
    if (one_cluster) {
        // a call of few units is one cluster: it joins its pieces itself, behind a
        // barrier that also orders their stores
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
        if (force_partial && blockIdx.x == 0 && threadIdx.x == 0) *pre.ready = 0;   // for a replay of this call
        for (size_t i = blockIdx.x; i < (size_t)items; i += gridDim.x) join_item<T, D>(kv, a, S::QR, i, o_part, ml_part, meta[i], pre, reinterpret_cast<float *>(psm));
    }
}

// query rows of an item: the n8 tiles that hold the group's rows, four at most
int paged_nt(int qg, int G) { return std::min(4, (qg * G + 7) / 8); }

struct Scratch {
    size_t items, slots, ml_at, meta_at, bytes;
};
Scratch scratch_of(int M, int qg, int n_heads, int n_kv, int D, int sm_count) {
    const int G = n_heads / n_kv, QR = paged_nt(qg, G) * 8;
    const size_t groups = (M + qg - 1) / qg, qts = ((size_t)qg * G + QR - 1) / QR;
    Scratch s;
    s.items = groups * n_kv * qts;
    s.slots = s.items + (size_t)sm_count * CTAS_PER_SM;
    s.ml_at = s.slots * QR * D * 4;
    s.meta_at = s.ml_at + ((s.slots * QR * 8 + 255) & ~(size_t)255);
    s.bytes = s.meta_at + s.items * sizeof(int2);
    return s;
}

template <typename T, int D, int NT>
cudaError_t launch_main(const PagedKV &kv, const PagedQuery &q, int key_begin, const PrefixPartials &pre, const Scratch &s,
                        char *ws, int grid, bool cluster, cudaStream_t st) {
    using P = PagedShape<D, NT>;
    static bool attr[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!attr[dev & 63]) {
        const cudaError_t e = cudaFuncSetAttribute(paged_attn_kernel<T, D, NT>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, P::SMEM);
        if (e != cudaSuccess) return e;
        attr[dev & 63] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(PT);
    cfg.dynamicSmemBytes = P::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = grid;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, paged_attn_kernel<T, D, NT>, kv, q, key_begin, pre.splits > 0 ? 1 : 0,
                              reinterpret_cast<float *>(ws), reinterpret_cast<float *>(ws + s.ml_at),
                              reinterpret_cast<int2 *>(ws + s.meta_at), pre, cluster ? 1 : 0, (int)s.items);
}

template <typename T, int D>
cudaError_t run(const PagedKV &kv, const PagedQuery &q, int key_begin, const PrefixPartials &pre, char *ws,
                int sm_count, cudaStream_t st) {
    const int G = q.n_heads / kv.n_kv, NT = paged_nt(q.qg, G);
    const Scratch s = scratch_of(q.M, q.qg, q.n_heads, kv.n_kv, D, sm_count);
    // no more CTAs than the table can hold units for: behind a prefix pass the ones
    // without a free SM would only start when the pass ends
    const int64_t cap = std::max(0, paged_capacity(kv) - key_begin);
    const int64_t units = (int64_t)s.items * ((cap + UNIT - 1) / UNIT + LEAD);
    // Beside a prefix pass that leaves SMs free, this kernel takes those and no more:
    // CTAs that had to wait for the pass would be the last.  That is for own keys that
    // are short beside the prefix, as prefix_splits says with both sides' times; with
    // long ones (which only the device knows) the SMs of the pass are missed.
    const int free_sms = pre.splits && pre.ctas <= sm_count - sm_count / 4 ? sm_count - pre.ctas : sm_count;
    // few units: one cluster that joins its own pieces, no second kernel (one row of
    // 300 keys, 8 / 2 heads of 64, 7.95 -> 7.2 us).  The host knows no lengths, so the
    // table's width decides: up to 1,856 keys for one row with two KV heads, 320 for
    // four rows.  A wider table takes the two kernels; back to back on the same inputs
    // that is one row 7.2 us either way, four rows 8.1 us here and 7.5 there.
    const bool cluster = units <= ONE_CLUSTER * CLUSTER_UNITS;
    const int grid = (int)std::min<int64_t>(cluster ? ONE_CLUSTER : (int64_t)free_sms * CTAS_PER_SM, units);
    cudaError_t e;
    switch (NT) {
        case 1: e = launch_main<T, D, 1>(kv, q, key_begin, pre, s, ws, grid, cluster, st); break;
        case 2: e = launch_main<T, D, 2>(kv, q, key_begin, pre, s, ws, grid, cluster, st); break;
        case 3: e = launch_main<T, D, 3>(kv, q, key_begin, pre, s, ws, grid, cluster, st); break;
        default: e = launch_main<T, D, 4>(kv, q, key_begin, pre, s, ws, grid, cluster, st); break;
    }
    if (e != cudaSuccess || cluster) return e;
    return launch_pdl(attn_join<T, D>, dim3((unsigned)s.items), dim3(256), 0, st, kv, q, NT * 8,
                      (const float *)ws, (const float *)(ws + s.ml_at), (const int2 *)(ws + s.meta_at), pre);
}

}  // namespace

size_t paged_attn_scratch(int M, int qg, int n_heads, int n_kv, int D, int sm_count) {
    return scratch_of(M, qg, n_heads, n_kv, D, sm_count).bytes;
}

cudaError_t paged_attn(const PagedKV &kv, const PagedQuery &q, int key_begin, const PrefixPartials &pre, void *scratch,
                       int sm_count, cudaStream_t st) {
    char *ws = static_cast<char *>(scratch);
    if (kv.D == 128)
        return kv.bf16 ? run<__nv_bfloat16, 128>(kv, q, key_begin, pre, ws, sm_count, st)
                       : run<__half, 128>(kv, q, key_begin, pre, ws, sm_count, st);
    return kv.bf16 ? run<__nv_bfloat16, 64>(kv, q, key_begin, pre, ws, sm_count, st)
                   : run<__half, 64>(kv, q, key_begin, pre, ws, sm_count, st);
}

}  // namespace mlxcat
