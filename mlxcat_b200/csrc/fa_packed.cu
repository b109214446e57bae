// fa_packed.cu -- attention on the 5th-generation tensor cores for many query
// rows: causal attention of packed prompts, and the pass of a whole batch over
// the keys of a shared prefix.
//
// CTA = up to two tiles of 128 query rows of one KV head.  A row is a (token,
// query head of the group) pair, token-major, so all G heads that share a KV
// head read its tiles once and a short sequence still fills rows.  Keys stream
// in blocks of 128 through a ring of shared-memory slots (K_0, V_0, K_1, ...).
// Per block j and tile i:
//   S_i  = Q_i K_j^T      tcgen05.mma, both operands from shared memory
//   P_i  = 2^(S_i c - m)  four softmax warps per tile, a thread per row; the
//                          reference m moves only when a row's maximum grows by
//                          more than 8 (log2 units), so P <= 256 fits fp16.  P
//                          goes back over the first half of S_i in TMEM.
//   O_i += P_i V_j        A = P_i from TMEM, B = V_j read in place as an
//                          MN-major operand
// The two tiles take turns: while the tensor cores work for one, the other's
// softmax runs (128 x 128 exponentials take the SM as long as the tile's two
// products).
//
// Keys past a sequence's end are never a factor: their scores are replaced
// (not added to), and the rows of V between the end and the next multiple of 16
// are zeroed in shared memory before the product, so what lies behind a
// sequence (another prompt, an unwritten page, NaN) does not reach it.
//
// Warps: 0 TMEM allocation and TMA producer, 1 and 2 issuers of the products with
// V of tiles 0 and 1, 3 and 12 issuers of their scores, 4-7 softmax of tile 0,
// 8-11 of tile 1.  Every wait is bounded; a timeout sets *err and an abort
// flag after which every role skips its work, the producer waits for its copies
// and the issuer for what it committed, and the CTA frees TMEM.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"
#include "tc.cuh"

namespace mlxcat {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn();

namespace {

constexpr int TM = 128;                 // query rows of a tile (MMA M)
constexpr int KB = 128;                 // keys of a block
constexpr int BOX = 128 * 128;          // [128 rows][64 features] swizzled
constexpr int KSLOTS = 2, VSLOTS = 3;   // rings of K and V blocks
constexpr int THREADS = 416;
constexpr int SB = 64;                  // keys of a score buffer: two per tile
constexpr uint32_t COL_S = 0, COL_O = 256;

enum PkErr { PK_Q = 61, PK_KV, PK_FREE, PK_S, PK_P, PK_PV, PK_ALIGN };

struct Bars {
    unsigned long long q_full, k_full[KSLOTS], k_free[KSLOTS], v_full[VSLOTS], v_free[VSLOTS], skew, tail, fin[4];
    unsigned long long s_full[2][2], p_full[2][2], pv_done[2][2];   // [tile][score buffer]
    uint32_t tmem;
    int abort;
};

template <int D>
struct Shape {
    static constexpr int HALVES = D / 64;
    static constexpr int TILE = HALVES * BOX;
    static constexpr int SMEM = (2 + KSLOTS + VSLOTS) * TILE + (int)sizeof(Bars);
    static_assert(SMEM <= 227 * 1024, "two Q tiles and the ring must fit one CTA");
};

struct Args {
    int prefix;                 // 0: packed sequences, 1: shared prefix
    const int32_t *cu_q, *cu_k; // packed
    int n_seq, causal, Tq, Tk;
    PagedKV kv;                 // prefix
    const int32_t *trow, *tpos;
    int M, prefix_len, splits;
    float *o_part, *ml_part;
    int Hq, Hkv, G, TQ;         // TQ tokens of G rows each fill a tile
    float scale_log2;
    void *out;
    int32_t *err;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}

// one lane of the warp, the same each time
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}\n" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float lo2(uint64_t x) { return __uint_as_float((uint32_t)x); }
__device__ __forceinline__ float hi2(uint64_t x) { return __uint_as_float((uint32_t)(x >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint64_t exp2_unit(uint64_t z) { return pack2(tc::ex2_approx(lo2(z)), tc::ex2_approx(hi2(z))); }

// 2^z on the FMA pipe for finite z <= 8: z = n + r, n the nearest integer (taken
// from the low bits of z + 1.5 * 2^23), 2^r by the polynomial 1 + r (c1 + ...) of
// least relative error on [-1/2, 1/2] (1.0e-4 at degree 3, 2.8e-6 at degree 4,
// fitted by reweighted least squares), n added to the exponent.  Below -126 the
// result is 2^-126.
template <int DEG>
__device__ __forceinline__ uint64_t exp2_poly(uint64_t z) {
    z = pack2(fmaxf(lo2(z), -126.f), fmaxf(hi2(z), -126.f));
    const uint64_t magic = pack2(12582912.f, 12582912.f), neg = pack2(-12582912.f, -12582912.f), minus = pack2(-1.f, -1.f);
    const uint64_t t = add2(z, magic), r = fma2(add2(t, neg), minus, z), one = pack2(1.f, 1.f);
    uint64_t p;
    if (DEG == 3) {
        p = fma2(r, pack2(0.055008933f, 0.055008933f), pack2(0.24221097f, 0.24221097f));
        p = fma2(p, r, pack2(0.6932829f, 0.6932829f));
    } else {
        p = fma2(r, pack2(0.009582853f, 0.009582853f), pack2(0.055906426f, 0.055906426f));
        p = fma2(p, r, pack2(0.24024099f, 0.24024099f));
        p = fma2(p, r, pack2(0.69312418f, 0.69312418f));
    }
    p = fma2(p, r, one);
    return pack2(__uint_as_float((uint32_t)p + ((uint32_t)t << 23)),
                 __uint_as_float((uint32_t)(p >> 32) + ((uint32_t)(t >> 32) << 23)));
}

// a whole 32-byte sector per thread: rows lie apart, so 16-byte stores would fill
// every sector twice
__device__ __forceinline__ void store32(void *p, const uint32_t *v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

template <typename T>
struct Pk;
template <>
struct Pk<__half> {
    static constexpr int POLY = 4, DEG = 4;   // pairs of 16 whose exponentials run on the FMA pipe
    static constexpr uint32_t fmt = 0;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};
template <>
struct Pk<__nv_bfloat16> {
    static constexpr int POLY = 4, DEG = 3;
    static constexpr uint32_t fmt = (1u << 7) | (1u << 10);   // A and B bf16
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};

// The whole warp waits for phase `n` of a barrier: false when it ran out of time
// or the CTA has been given up.
__device__ __forceinline__ bool wait_all(unsigned long long &bar, int n, volatile int *abort, int32_t *err, int code) {
    const uint32_t b = tc::smem_u32(&bar);
    const bool r = tc::mbar_try_wait(b, n & 1) || tc::mbar_wait_abort(b, n & 1, abort, err, code);
    return __all_sync(0xffffffffu, r);
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1)
fa_packed_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                 const __grid_constant__ CUtensorMap vmap, const Args a) {
    using S = Shape<D>;
    // no static shared memory in this kernel: the dynamic block starts on a
    // 1024-byte boundary, as the swizzled tiles need (checked, there is no room to shift)
    extern __shared__ __align__(1024) unsigned char sm[];
    if (tc::smem_u32(sm) & 1023) {
        if (a.err) atomicExch(a.err, PK_ALIGN);
        return;
    }
    unsigned char *sm_q = sm, *sm_k = sm + 2 * S::TILE, *sm_v = sm_k + KSLOTS * S::TILE;
    Bars &fb = *reinterpret_cast<Bars *>(sm_v + VSLOTS * S::TILE);
    volatile int *abort = &fb.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // the kernel that follows a prefix pass starts on the SMs that this one leaves
    // free, without waiting for it: so the pass's own predecessor must be done first
    griddep_wait();
    griddep_launch_dependents();

    // ---- which tokens and keys: tokens [tok0, tok0 + ntok) of the packed
    // queries, keys [kbeg, kend) counted from the sequence's start
    const int h = blockIdx.x % a.Hkv;
    int tok0 = 0, ntok = 0, kbeg = 0, kend = 0, krow0 = 0, first_lim = 0, split = 0;
    if (!a.prefix) {
        // sequence s owns tile numbers from cu_q[s] / (2 TQ) + s on: one more than
        // its tokens need at most, so the map needs no prefix sum
        const int tile = gridDim.x / a.Hkv - 1 - blockIdx.x / a.Hkv;   // the last tiles see most keys: first
        int lo = 0, hi = a.n_seq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (__ldg(a.cu_q + mid) / (2 * a.TQ) + mid <= tile) lo = mid;
            else hi = mid - 1;
        }
        // offsets outside the buffers are cut to them
        const int q0 = min(max(__ldg(a.cu_q + lo), 0), a.Tq), q1 = min(max(__ldg(a.cu_q + lo + 1), q0), a.Tq);
        const int k0 = min(max(__ldg(a.cu_k + lo), 0), a.Tk), k1 = min(max(__ldg(a.cu_k + lo + 1), k0), a.Tk);
        const int at = (tile - (__ldg(a.cu_q + lo) / (2 * a.TQ) + lo)) * 2 * a.TQ;   // token of the sequence
        if (at >= 0 && at < q1 - q0) {
            tok0 = q0 + at;
            ntok = min(2 * a.TQ, q1 - tok0);
        }
        krow0 = k0;
        const int nk = k1 - k0, nq = q1 - q0;
        first_lim = a.causal ? nk - nq + at : nk - 1;
        kend = a.causal ? min(nk, first_lim + ntok) : nk;   // one past the last key any row sees
    } else {
        const int pairs = (a.M + 2 * a.TQ - 1) / (2 * a.TQ), x = blockIdx.x / a.Hkv;
        split = x / pairs;
        tok0 = (x % pairs) * 2 * a.TQ;
        ntok = min(2 * a.TQ, a.M - tok0);
        const int blocks = (a.prefix_len + KB - 1) / KB;
        kbeg = (int)((int64_t)blocks * split / a.splits) * KB;
        kend = min(a.prefix_len, (int)((int64_t)blocks * (split + 1) / a.splits) * KB);
    }
    const bool any = ntok > 0;
    const int nb = any && kend > kbeg ? (kend - kbeg + KB - 1) / KB : 0;
    const int ns = nb ? (kend - kbeg + SB - 1) / SB : 0;   // score blocks
    const int tiles = ntok > a.TQ ? 2 : 1;

    if (threadIdx.x == 0) {
        tc::mbar_init(tc::smem_u32(&fb.q_full), 1);
        tc::mbar_init(tc::smem_u32(&fb.skew), 1);
        tc::mbar_init(tc::smem_u32(&fb.tail), 1);
        for (int s = 0; s < KSLOTS; ++s) {
            tc::mbar_init(tc::smem_u32(&fb.k_full[s]), 1);
            tc::mbar_init(tc::smem_u32(&fb.k_free[s]), tiles);   // each tile's score issuer
        }
        for (int s = 0; s < VSLOTS; ++s) {
            tc::mbar_init(tc::smem_u32(&fb.v_full[s]), 1);
            tc::mbar_init(tc::smem_u32(&fb.v_free[s]), tiles);   // each tile's value issuer
        }
        for (int i = 0; i < 2; ++i) {
            for (int b = 0; b < 2; ++b) {
                tc::mbar_init(tc::smem_u32(&fb.s_full[i][b]), 1);
                tc::mbar_init(tc::smem_u32(&fb.p_full[i][b]), 4);   // the tile's softmax warps
                tc::mbar_init(tc::smem_u32(&fb.pv_done[i][b]), 1);
            }
            tc::mbar_init(tc::smem_u32(&fb.fin[i]), 1);
            tc::mbar_init(tc::smem_u32(&fb.fin[2 + i]), 1);
        }
        fb.abort = 0;
        tc::fence_barrier_init();
        tc::prefetch_tmap(&qmap);
        tc::prefetch_tmap(&kmap);
        tc::prefetch_tmap(&vmap);
    }
    if (warp == 0 && nb) tc::tmem_alloc(tc::smem_u32(&fb.tmem), 512);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = fb.tmem;

    if (warp == 0 && nb) {
        // ---------------- TMA producer ----------------
        if (lane == 0) {
            const uint32_t qb = tc::smem_u32(&fb.q_full);
            tc::mbar_arrive_expect_tx(qb, (uint32_t)(tiles * S::HALVES * a.G * a.TQ * 128));
            for (int i = 0; i < tiles; ++i)
                for (int x = 0; x < S::HALVES; ++x)
                    tc::tma_load_3d(tc::smem_u32(sm_q + i * S::TILE + x * BOX), &qmap, x * 64, h * a.G, tok0 + i * a.TQ, qb);
        }
        // boxes of a block: `bt` tokens each (a page, or all 128 keys)
        const int bt = a.prefix ? min(KB, 1 << a.kv.page_shift) : KB, nbox = KB / bt;
        const int32_t *table = nullptr;
        if (a.prefix) {
            // any row's table will do: the first token's that is no padding
            int row = -1;
            for (int m0 = 0; m0 < a.M && row < 0; m0 += 32) {
                const int r = m0 + lane < a.M ? __ldg(a.trow + m0 + lane) : -1;
                const unsigned ok = __ballot_sync(0xffffffffu, r >= 0 && r < a.kv.rows);
                if (ok) row = __shfl_sync(0xffffffffu, r, __ffs(ok) - 1);
            }
            table = row < 0 ? nullptr : a.kv.table + (size_t)row * a.kv.max_pages;
        }
        int issued = 0;
        bool ok = true;
        for (int f = 0; f < 2 * nb && ok; ++f) {   // K_0, V_0, K_1, ...
            const int j = f >> 1, v = f & 1, s = v ? j % VSLOTS : j % KSLOTS, turn = v ? j / VSLOTS : j / KSLOTS;
            if (turn) ok = wait_all(v ? fb.v_free[s] : fb.k_free[s], turn - 1, abort, a.err, PK_FREE);
            if (!ok) break;
            const CUtensorMap *map = v ? &vmap : &kmap;
            const uint32_t bar = tc::smem_u32(v ? &fb.v_full[s] : &fb.k_full[s]);
            const uint32_t dst = tc::smem_u32((v ? sm_v : sm_k) + s * S::TILE);
            const int key0 = kbeg + j * KB;
            const int boxes = a.prefix ? min(nbox, (kend - key0 + bt - 1) / bt) : 1;
            if (lane == 0) tc::mbar_arrive_expect_tx(bar, (uint32_t)(boxes * S::HALVES * bt * 128));
            __syncwarp();
            if (lane < boxes * S::HALVES) {
                const int b = lane / S::HALVES, x = lane % S::HALVES;
                if (a.prefix) {
                    const int key = key0 + b * bt;
                    int page = table ? __ldg(table + (key >> a.kv.page_shift)) : -1;
                    if (page < 0 || page >= a.kv.n_pages) {   // reads as zeros (a box outside the tensor)
                        if (table && a.err) atomicExch(a.err, PE_PAGE);
                        page = a.kv.n_pages;
                    }
                    tma_load_4d(dst + x * BOX + b * bt * 128, map, x * 64, key & ((1 << a.kv.page_shift) - 1), h, page, bar);
                } else {
                    tma_load_4d(dst + x * BOX, map, x * 64, krow0 + key0, h, 0, bar);
                }
            }
            issued = f + 1;
        }
        // the last block ends inside 16 keys: zero the rows of V behind its last key
        const int nv = kend - kbeg - (nb - 1) * KB, sl = (nb - 1) % VSLOTS;
        if (ok && (nv & 15) && wait_all(fb.v_full[sl], (nb - 1) / VSLOTS, abort, a.err, PK_KV)) {
            unsigned char *v = sm_v + sl * S::TILE + nv * 128;
            const int words = (16 - (nv & 15)) * 8;
            for (int w = lane; w < words * S::HALVES; w += 32)
                *reinterpret_cast<uint4 *>(v + (w / words) * BOX + (w % words) * 16) = make_uint4(0, 0, 0, 0);
            tc::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(tc::smem_u32(&fb.tail));
        }
        // copies in flight must land before the CTA's shared memory is released
        if (lane == 0) {
            tc::mbar_wait(tc::smem_u32(&fb.q_full), 0, nullptr, 0);
            for (int f = max(0, issued - 2 * VSLOTS); f < issued; ++f) {
                const int j = f >> 1, v = f & 1;
                if (!v && j + KSLOTS < (issued + 1) / 2) continue;   // filled again since
                tc::mbar_wait(tc::smem_u32(v ? &fb.v_full[j % VSLOTS] : &fb.k_full[j % KSLOTS]), (v ? j / VSLOTS : j / KSLOTS) & 1, nullptr, 0);
            }
        }
    } else if ((warp == 3 || warp == 12) && nb && (warp == 3 || tiles == 2)) {
        // ---------------- issuer of tile i's scores (the whole warp waits, one lane issues) ----------------
        // Issuing, committing and waiting take as long as the products themselves: every
        // chain of products has a warp of its own.
        constexpr uint32_t idesc_s = tc::idesc_f16_f32(TM, SB) | Pk<T>::fmt;
        const int i = warp == 3 ? 0 : 1;
        // descriptors differ only in their address field (16-byte units)
        const uint64_t qd = tc::sdesc_k_sw128(tc::smem_u32(sm_q + i * S::TILE)), kd0 = tc::sdesc_k_sw128(tc::smem_u32(sm_k));
        const uint32_t tS = tmem + COL_S + i * 128;
        bool ok = wait_all(fb.q_full, 0, abort, a.err, PK_Q);
        // tile 1 starts when tile 0 is through its first scores, so that the one's
        // softmax meets the other's products from then on
        if (i) ok = ok && wait_all(fb.skew, 0, abort, a.err, PK_P);
        // keys 64 n .. 64 n + 63 into buffer n & 1
        for (int n = 0; n < ns && ok; ++n) {
            const int b = n & 1, j = n >> 1, sl = j % KSLOTS;
            if (!b) ok = wait_all(fb.k_full[sl], j / KSLOTS, abort, a.err, PK_KV);
            // the scores lie over P of block n - 2: the product that reads it comes first
            if (n >= 2) ok = ok && wait_all(fb.pv_done[i][b], j - 1, abort, a.err, PK_PV);
            if (!ok) break;
            tc::fence_after_sync();
            const uint64_t kd = kd0 + (uint32_t)(sl * (S::TILE >> 4) + b * (SB * 128 >> 4));
            const uint32_t d = tS + b * SB;
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    const uint32_t off = (uint32_t)(((kk >> 2) * BOX + (kk & 3) * 32) >> 4);
                    tc::mma_ss_f16(d, qd + off, kd + off, idesc_s, kk ? 1u : 0u);
                }
                tc::mma_commit(tc::smem_u32(&fb.s_full[i][b]));
                if (b) tc::mma_commit(tc::smem_u32(&fb.k_free[sl]));
            }
            __syncwarp();
        }
        // everything issued must finish before TMEM is freed
        if (elect_one()) tc::mma_commit(tc::smem_u32(&fb.fin[2 + i]));
        __syncwarp();
        tc::mbar_wait(tc::smem_u32(&fb.fin[2 + i]), 0, nullptr, 0);
    } else if ((warp == 1 || warp == 2) && nb && warp <= tiles) {
        // ---------------- issuer of tile i's O += P V ----------------
        constexpr uint32_t idesc_pv = tc::idesc_f16_f32(TM, D) | (1u << 16) | Pk<T>::fmt;   // B (V) MN-major
        const int i = warp - 1;
        const uint64_t vd0 = tc::sdesc_mn_sw128(tc::smem_u32(sm_v), BOX);
        const uint32_t tS = tmem + COL_S + i * 128, tO = tmem + COL_O + i * 128;
        bool ok = true;
        for (int n = 0; n < ns && ok; ++n) {
            const int b = n & 1, j = n >> 1, sl = j % VSLOTS;
            const uint64_t vd = vd0 + (uint32_t)(sl * (S::TILE >> 4) + b * (SB * 128 >> 4));
            const int nv = n + 1 < ns ? SB : kend - kbeg - n * SB, ks = (nv + 15) / 16;   // 16-key steps that hold keys
            if (!b) ok = wait_all(fb.v_full[sl], j / VSLOTS, abort, a.err, PK_KV);
            if (nv & 15) ok = ok && wait_all(fb.tail, 0, abort, a.err, PK_KV);   // the rows behind the last key are zeroed
            ok = ok && wait_all(fb.p_full[i][b], j, abort, a.err, PK_P);
            if (!ok) break;
            tc::fence_after_sync();
            if (elect_one()) {
                if (ks == SB / 16) {
#pragma unroll
                    for (int kk = 0; kk < SB / 16; ++kk)
                        tc::mma_ts_f16(tO, tS + b * SB + kk * 8, vd + kk * 128, idesc_pv, (n | kk) ? 1u : 0u);
                } else {
                    for (int kk = 0; kk < ks; ++kk)
                        tc::mma_ts_f16(tO, tS + b * SB + kk * 8, vd + kk * 128, idesc_pv, (n | kk) ? 1u : 0u);
                }
                tc::mma_commit(tc::smem_u32(&fb.pv_done[i][b]));
                if (b) tc::mma_commit(tc::smem_u32(&fb.v_free[sl]));   // the block's V is no longer needed here
            }
            __syncwarp();
        }
        if (elect_one()) tc::mma_commit(tc::smem_u32(&fb.fin[i]));
        __syncwarp();
        tc::mbar_wait(tc::smem_u32(&fb.fin[i]), 0, nullptr, 0);
    } else if (warp >= 4 && warp < 12 && any) {
        // ---------------- softmax and epilogue: thread = query row ----------------
        const int i = (warp - 4) >> 2, quarter = warp & 3;
        if (i < tiles) {
            const int r = quarter * 32 + lane, j0 = r / a.G;     // row of the tile, token of the tile
            const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
            const int tk = i * a.TQ + j0;                          // token of the CTA
            const bool valid = r < a.G * a.TQ && tk < ntok;
            int lim = -1;                                          // last key the row sees
            bool pad = !valid;
            if (valid) {
                if (!a.prefix) lim = a.causal ? min(first_lim + tk, kend - 1) : kend - 1;
                else if (__ldg(a.trow + tok0 + tk) >= 0) lim = min(__ldg(a.tpos + tok0 + tk), kend - 1);
                else pad = true;
            }
            lim = pad ? 0x3fffffff : lim - kbeg;   // rows nobody reads need no mask
            float m_used = -INFINITY, l = 0.f;
            bool ok = true;
            const uint32_t tS = tmem + lane_base + COL_S + i * 128, tO = tmem + lane_base + COL_O + i * 128;
            const uint64_t sc2 = pack2(a.scale_log2, a.scale_log2);
            for (int n = 0; n < ns; ++n) {
                const int b = n & 1;
                ok = wait_all(fb.s_full[i][b], n >> 1, abort, a.err, PK_S);
                if (!ok) break;
                tc::fence_after_sync();
                uint32_t v[SB];
                tc::tmem_ld32(tS + b * SB, v);
                tc::tmem_ld32(tS + b * SB + 32, v + 32);
                tc::tmem_wait_ld();
                const int rel = lim - n * SB;   // columns 0..rel are seen
                const bool full = __all_sync(0xffffffffu, rel >= SB - 1);
                if (!full) {
#pragma unroll
                    for (int x = 0; x < SB; ++x)
                        if (x > rel) v[x] = 0xff800000u;   // -inf
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int x = 0; x < SB; x += 2)
                    mx4[(x >> 1) & 3] = max3_nan(mx4[(x >> 1) & 3], __uint_as_float(v[x]), __uint_as_float(v[x + 1]));
                const float mx = max3_nan(max3_nan(mx4[0], mx4[1], mx4[2]), mx4[3], mx4[3]) * a.scale_log2;
                float alpha = 1.f;
                if (mx > m_used + 8.f) {
                    alpha = m_used == -INFINITY ? 0.f : tc::ex2_approx(m_used - mx);
                    m_used = mx;
                }
                // a row whose reference moved scales its O once the last product is in
                if (n && __any_sync(0xffffffffu, alpha != 1.f)) {
                    ok = wait_all(fb.pv_done[i][b ^ 1], (n - 1) >> 1, abort, a.err, PK_PV);
                    if (!ok) break;
                    tc::fence_after_sync();
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16];
                        tc::tmem_ld16(tO + c * 16, o);
                        tc::tmem_wait_ld();
#pragma unroll
                        for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
                        tc::tmem_st16(tO + c * 16, o);
                    }
                }
                const float nm = m_used == -INFINITY ? 0.f : -m_used;
                const uint64_t nm2 = pack2(nm, nm);
                uint64_t sum2[2] = {0, 0};
                uint32_t p[SB / 2];
#pragma unroll
                for (int x = 0; x < SB / 2; ++x) {
                    const uint64_t z = fma2(pack2(__uint_as_float(v[2 * x]), __uint_as_float(v[2 * x + 1])), sc2, nm2);
                    const uint64_t e = exp2_unit(z);
                    sum2[x & 1] = add2(sum2[x & 1], e);
                    p[x] = Pk<T>::pack(lo2(e), hi2(e));
                }
                tc::tmem_st32(tS + b * SB, p);
                tc::tmem_wait_st();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(tc::smem_u32(&fb.p_full[i][b]));
                if (n == 0 && warp == 4 && lane == 0) tc::mbar_arrive(tc::smem_u32(&fb.skew));
                sum2[0] = add2(sum2[0], sum2[1]);
                l = l * alpha + (lo2(sum2[0]) + hi2(sum2[0]));
            }
            if (ok && nb) {
                ok = wait_all(fb.pv_done[i][(ns - 1) & 1], (ns - 1) >> 1, abort, a.err, PK_PV) && !*abort;
                ok = __all_sync(0xffffffffu, ok);
                tc::fence_after_sync();
            }
            if (ok) {
                const int gh = r - j0 * a.G;
                const float inv = l != 0.f ? 1.f / l : 0.f;
                const bool wide = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
                T *dst = reinterpret_cast<T *>(a.out) + ((size_t)(tok0 + tk) * a.Hq + h * a.G + gh) * D;
                const size_t prow = ((size_t)split * a.Hkv + h) * ((size_t)a.M * a.G) + (size_t)(tok0 + tk) * a.G + gh;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t acc[32];
                    __syncwarp();
                    if (nb) {
                        tc::tmem_ld32(tO + c * 32, acc);
                        tc::tmem_wait_ld();
                    }
                    const bool live = nb && l != 0.f;
#pragma unroll
                    for (int x = 0; x < 32; ++x)
                        if (!live) acc[x] = 0u;
                    if (!pad && a.prefix) {
                        float *p = a.o_part + prow * D + c * 32;
#pragma unroll
                        for (int x = 0; x < 4; ++x) store32(p + x * 8, acc + x * 8);
                    } else if (!pad) {
                        uint32_t y[16];
#pragma unroll
                        for (int x = 0; x < 16; ++x)
                            y[x] = Pk<T>::pack(__uint_as_float(acc[2 * x]) * inv, __uint_as_float(acc[2 * x + 1]) * inv);
                        if (wide) {
                            store32(dst + c * 32, y);
                            store32(dst + c * 32 + 16, y + 8);
                        } else {
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                reinterpret_cast<uint4 *>(dst + c * 32)[x] = make_uint4(y[4 * x], y[4 * x + 1], y[4 * x + 2], y[4 * x + 3]);
                        }
                    }
                }
                if (a.prefix && !pad) *reinterpret_cast<float2 *>(a.ml_part + prow * 2) = make_float2(m_used, l);
            }
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 0 && nb) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, 512);
    }
}

// [pages][heads][tokens][D] with strides (elements); a box is 64 features of `box_tokens` tokens
bool kv_map(CUtensorMap *m, const void *base, bool bf16, int D, uint64_t tokens, uint64_t heads, uint64_t pages,
            int64_t token_stride, int64_t head_stride, int64_t page_stride, int box_tokens) {
    auto fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)D, tokens, heads, pages};
    const cuuint64_t strides[3] = {(cuuint64_t)token_stride * 2, (cuuint64_t)head_stride * 2, (cuuint64_t)page_stride * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)box_tokens, 1, 1};
    const cuuint32_t es[4] = {1, 1, 1, 1};
    return fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(base),
              dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool q_map(CUtensorMap *m, const void *base, bool bf16, int D, int heads, int tokens, int64_t token_stride, int G, int TQ) {
    auto fn = encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)token_stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)TQ};
    const cuuint32_t es[3] = {1, 1, 1};
    return fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base),
              dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
cudaError_t launch(const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, const Args &a, int64_t grid,
                   cudaStream_t st) {
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    static bool attr[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!attr[dev & 63]) {
        const cudaError_t e = cudaFuncSetAttribute(fa_packed_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   Shape<D>::SMEM);
        if (e != cudaSuccess) return e;
        attr[dev & 63] = true;
    }
    return launch_pdl(fa_packed_kernel<T, D>, dim3((unsigned)grid), dim3(THREADS), (size_t)Shape<D>::SMEM, st, q, k, v, a);
}

cudaError_t launch_any(const CUtensorMap &q, const CUtensorMap &k, const CUtensorMap &v, const Args &a, int D, bool bf16,
                       int64_t grid, cudaStream_t st) {
    if (D == 128)
        return bf16 ? launch<__nv_bfloat16, 128>(q, k, v, a, grid, st) : launch<__half, 128>(q, k, v, a, grid, st);
    return bf16 ? launch<__nv_bfloat16, 64>(q, k, v, a, grid, st) : launch<__half, 64>(q, k, v, a, grid, st);
}

}  // namespace

cudaError_t packed_attn(const PackedAttn &p, cudaStream_t st) {
    Args a = {};
    a.cu_q = p.cu_q; a.cu_k = p.cu_k;
    a.n_seq = p.n_seq; a.causal = p.causal; a.Tq = p.Tq; a.Tk = p.Tk;
    a.Hq = p.n_heads; a.Hkv = p.n_kv; a.G = p.n_heads / p.n_kv; a.TQ = TM / a.G;
    a.scale_log2 = p.scale_log2; a.out = p.out; a.err = p.err;
    CUtensorMap qm, km, vm;
    if (!q_map(&qm, p.q, p.bf16, p.D, p.n_heads, p.Tq, p.q_stride, a.G, a.TQ) ||
        !kv_map(&km, p.k, p.bf16, p.D, p.Tk, p.n_kv, 1, p.k_stride, p.D, p.k_stride, KB) ||
        !kv_map(&vm, p.v, p.bf16, p.D, p.Tk, p.n_kv, 1, p.v_stride, p.D, p.v_stride, KB))
        return cudaErrorInvalidValue;
    const int64_t tiles = (int64_t)p.Tq / (2 * a.TQ) + p.n_seq;
    return launch_any(qm, km, vm, a, p.D, p.bf16, tiles * p.n_kv, st);
}

int prefix_splits(int M, int n_heads, int n_kv, int prefix_len, int sm_count) {
    const int G = n_heads / n_kv, TQ = TM / G;
    const int64_t items = (int64_t)((M + 2 * TQ - 1) / (2 * TQ)) * n_kv;
    const int blocks = (prefix_len + KB - 1) / KB;
    // one wave of CTAs, two key blocks each at least
    return (int)std::max<int64_t>(1, std::min<int64_t>(sm_count / items, (blocks + 1) / 2));
}

cudaError_t prefix_attn(const PagedKV &kv, const PagedQuery &q, int prefix_len, const PrefixPartials &part, cudaStream_t st) {
    Args a = {};
    a.prefix = 1; a.kv = kv; a.trow = q.trow; a.tpos = q.tpos; a.M = q.M; a.prefix_len = prefix_len; a.splits = part.splits;
    a.o_part = part.o; a.ml_part = part.ml;
    a.Hq = q.n_heads; a.Hkv = kv.n_kv; a.G = q.n_heads / kv.n_kv; a.TQ = TM / a.G;
    a.scale_log2 = q.scale_log2; a.err = q.err;
    CUtensorMap qm, km, vm;
    const int ps = 1 << kv.page_shift, bt = std::min(KB, ps);
    if (!q_map(&qm, q.q, kv.bf16, kv.D, q.n_heads, q.M, (int64_t)q.n_heads * kv.D, a.G, a.TQ) ||
        !kv_map(&km, kv.k, kv.bf16, kv.D, ps, kv.n_kv, kv.n_pages, kv.token_stride, kv.head_stride, kv.page_stride, bt) ||
        !kv_map(&vm, kv.v, kv.bf16, kv.D, ps, kv.n_kv, kv.n_pages, kv.token_stride, kv.head_stride, kv.page_stride, bt))
        return cudaErrorInvalidValue;
    const int64_t pairs = (q.M + 2 * a.TQ - 1) / (2 * a.TQ);
    return launch_any(qm, km, vm, a, kv.D, kv.bf16, pairs * kv.n_kv * part.splits, st);
}

}  // namespace mlxcat
