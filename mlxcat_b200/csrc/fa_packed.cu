// fa_packed.cu -- attention on the 5th-generation tensor cores for many query
// rows: causal attention of packed prompts, and the pass of a whole batch over
// the keys of a shared prefix.
//
// Item of work = up to two tiles of 128 query rows of one KV head; a CTA takes one
// after the other (the next one's number comes from cluster launch control: a CTA
// that would have started later is cancelled and its item done here), so that the
// start of an item overlaps the end of the one before.  A row is a (token,
// query head of the group) pair, token-major, so all G heads that share a KV
// head read its tiles once and a short sequence still fills rows.  Keys stream
// in blocks of 128 through a ring of K and one of V; scores are formed 64 keys at
// a time into two buffers a tile, so that the next ones are there when a softmax
// ends.  Per 64 keys j and tile i:
//   S_i  = Q_i K_j^T      tcgen05.mma, both operands from shared memory
//   P_i  = 2^(S_i c - m)  four softmax warps per tile, a thread per row; the
//                          reference m moves only when a row's maximum grows by
//                          more than 8 (log2 units), so P <= 256 fits fp16.  P
//                          goes back over the first half of its S buffer in TMEM.
//                          It is rounded to the operands' 16 bits once, the sum of the
//                          row is taken of the unrounded values in fp32.  A second part
//                          would be a second product: the errors against 64 bits are
//                          at most 1.4 times those of an fp32 P (fp16 2.3e-4 to 2.9e-4
//                          against 2.0e-4, bf16 2.0e-3 to 2.4e-3 against 1.7e-3), and
//                          an fp16 weight below 2^-25 of the reference vanishes.
//   O_i += P_i V_j        A = P_i from TMEM, B = V_j read in place as an
//                          MN-major operand
// The two tiles take turns: while the tensor cores work for one, the other's
// softmax runs.
//
// Keys past a sequence's end are never a factor: their scores are replaced
// (not added to), and the rows of V between the end and the next multiple of 16
// are zeroed in shared memory before the product, so what lies behind a
// sequence (another prompt, an unwritten page, NaN) does not reach it.
//
// Measured on B200s (32 query, 8 KV heads of 128): three prompts of 2,045 to
// 6,144 tokens 551 to 558 us, 1.07 PFLOP/s of visible pairs (496 us, 1.20 in single
// launches before the power limit lowers the clock); sixteen of 33 to 1,500 tokens
// 226 to 229 us.
// A block of 64 keys takes a tile 1,650 cycles: its softmax 1,400 (the
// exponentials of both tiles share 16 units, 1,024 cycles), the products of both
// tiles about 1,500 (an MMA of 64 or 128 columns takes 58 to 65 cycles alike).  One
// score buffer of 128 keys a tile had half the score MMAs but made the chain score
// -> softmax -> product -> score the limit: 640 us; one issuing warp for all, 720;
// part of the exponentials as a polynomial on the FMA pipe, 3 to 5 % slower.
// Between items a tile pauses about 5,000 cycles (last product, output, new queries).
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
constexpr int FEW_BLOCKS = 8;           // key blocks a CTA of a prefix pass below which it takes half the SMs
constexpr int SB = 64;                  // keys of a score buffer: two per tile
constexpr uint32_t COL_S = 0, COL_O = 256;

enum PkErr { PK_Q = 61, PK_KV, PK_FREE, PK_S, PK_P, PK_PV, PK_ALIGN, PK_WORK };

// One item of work: up to two tiles of query tokens [tok0, tok0 + ntok) of KV head
// h against keys [kbeg, kend) of a sequence (counted from its start).
struct Work {
    int end;                    // no more items
    int tok0, ntok, kbeg, kend, krow0, first_lim, split, h;
    int nb, ns, tiles;          // key blocks, score blocks, tiles
};

struct Bars {
    unsigned long long q_full[2], q_free[2], k_full[KSLOTS], k_free[KSLOTS], v_full[VSLOTS], v_free[VSLOTS];
    unsigned long long s_full[2][2], p_full[2][2], pv_done[2][2];   // [tile][score buffer]
    unsigned long long o_free[2], work_full[2], work_free[2], next, v_part, skew, fin[4];
    __align__(16) uint32_t response[4];   // of the request for the next item
    Work work[2];
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
    unsigned long long *ready, token;   // the sign for the kernel beside the pass
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
__device__ __forceinline__ uint64_t exp2_2(uint64_t z) { return pack2(tc::ex2_approx(lo2(z)), tc::ex2_approx(hi2(z))); }

// a whole 32-byte sector per thread: rows lie apart, so 16-byte stores would fill
// every sector twice
__device__ __forceinline__ void store32(void *p, const uint32_t *v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}

__device__ __forceinline__ void prefetch_3d(const CUtensorMap *map, int x, int y, int z) {
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];\n" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x),
                 "r"(y), "r"(z) : "memory");
}

template <typename T>
struct Pk;
template <>
struct Pk<__half> {
    static constexpr uint32_t fmt = 0;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};
template <>
struct Pk<__nv_bfloat16> {
    static constexpr uint32_t fmt = (1u << 7) | (1u << 10);   // A and B bf16
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
};

// Ask the launch for a CTA that has not started (cluster launch control): it will
// not start, and its number arrives in 16 bytes of shared memory.
__device__ __forceinline__ void request_next(uint32_t response, uint32_t bar) {
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n" ::"r"(response), "r"(bar)
                 : "memory");
}
// false: every CTA has started
__device__ __forceinline__ bool next_item(uint32_t response, int *id) {
    uint32_t got, x;
    asm volatile(
        "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
        "ld.shared.b128 r, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}\n"
        : "=r"(got), "=r"(x)
        : "r"(response)
        : "memory");
    if (got) *id = (int)x;
    // the response is written again by the async proxy
    tc::fence_proxy_async_smem();
    return got != 0;
}

// Item `id` of the grid, for a whole warp; ntok <= 0: none there.
__device__ __forceinline__ Work work_of(const Args &a, int id) {
    Work w = {};
    w.h = id % a.Hkv;
    const int x = id / a.Hkv;
    if (!a.prefix) {
        // sequence s owns tile numbers from cu_q[s] / (2 TQ) + s on: one more than
        // its tokens need at most, so the map needs no prefix sum
        const int tile = gridDim.x / a.Hkv - 1 - x;   // the last tiles see most keys: first
        // the last sequence that starts at or before it, 32 probes at a time; the last
        // round's loads bring the sequence's bounds along
        const int lane = threadIdx.x & 31;
        int lo = 0, n = a.n_seq;
        while (n > 32) {
            const int step = (n + 31) / 32, at = lo + lane * step;
            const bool in = lane * step < n && load_id(a.cu_q + at) / (2 * a.TQ) + at <= tile;
            const int k = max(__popc(__ballot_sync(0xffffffffu, in)) - 1, 0);
            lo += k * step;
            n = min(step, n - k * step);
        }
        int c[4] = {0, 0, 0, 0};
        if (lane < n) {
            c[0] = load_id(a.cu_q + lo + lane);
            c[1] = load_id(a.cu_q + lo + lane + 1);
            c[2] = load_id(a.cu_k + lo + lane);
            c[3] = load_id(a.cu_k + lo + lane + 1);
        }
        const int k = max(__popc(__ballot_sync(0xffffffffu, lane < n && c[0] / (2 * a.TQ) + lo + lane <= tile)) - 1, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = __shfl_sync(0xffffffffu, c[i], k);
        // offsets outside the buffers are cut to them
        const int q0 = min(max(c[0], 0), a.Tq), q1 = min(max(c[1], q0), a.Tq);
        const int k0 = min(max(c[2], 0), a.Tk), k1 = min(max(c[3], k0), a.Tk);
        const int at = (tile - (c[0] / (2 * a.TQ) + lo + k)) * 2 * a.TQ;   // token of the sequence
        if (at >= 0 && at < q1 - q0) {
            w.tok0 = q0 + at;
            w.ntok = min(2 * a.TQ, q1 - w.tok0);
        }
        w.krow0 = k0;
        const int nk = k1 - k0, nq = q1 - q0;
        w.first_lim = a.causal ? nk - nq + at : nk - 1;
        w.kend = a.causal ? min(nk, w.first_lim + w.ntok) : nk;   // one past the last key any row sees
    } else {
        const int pairs = (a.M + 2 * a.TQ - 1) / (2 * a.TQ);
        w.split = x / pairs;
        w.tok0 = (x % pairs) * 2 * a.TQ;
        w.ntok = min(2 * a.TQ, a.M - w.tok0);
        const int blocks = (a.prefix_len + KB - 1) / KB;
        w.kbeg = (int)((int64_t)blocks * w.split / a.splits) * KB;
        w.kend = min(a.prefix_len, (int)((int64_t)blocks * (w.split + 1) / a.splits) * KB);
    }
    if (w.ntok > 0 && w.kend > w.kbeg) {
        w.nb = (w.kend - w.kbeg + KB - 1) / KB;
        w.ns = (w.kend - w.kbeg + SB - 1) / SB;
    }
    w.tiles = w.ntok > a.TQ ? 2 : 1;
    return w;
}

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

    if (threadIdx.x == 0) {
        for (int s = 0; s < KSLOTS; ++s) {
            tc::mbar_init(tc::smem_u32(&fb.k_full[s]), 1);
            tc::mbar_init(tc::smem_u32(&fb.k_free[s]), 2);   // each tile's score issuer
        }
        for (int s = 0; s < VSLOTS; ++s) {
            tc::mbar_init(tc::smem_u32(&fb.v_full[s]), 1);
            tc::mbar_init(tc::smem_u32(&fb.v_free[s]), 2);   // each tile's value issuer
        }
        for (int i = 0; i < 2; ++i) {
            for (int b = 0; b < 2; ++b) {
                tc::mbar_init(tc::smem_u32(&fb.s_full[i][b]), 1);
                tc::mbar_init(tc::smem_u32(&fb.p_full[i][b]), 4);   // the tile's softmax warps
                tc::mbar_init(tc::smem_u32(&fb.pv_done[i][b]), 1);
            }
            tc::mbar_init(tc::smem_u32(&fb.q_full[i]), 1);
            tc::mbar_init(tc::smem_u32(&fb.q_free[i]), 1);
            tc::mbar_init(tc::smem_u32(&fb.o_free[i]), 4);
            tc::mbar_init(tc::smem_u32(&fb.work_full[i]), 1);
            tc::mbar_init(tc::smem_u32(&fb.work_free[i]), 12);      // every warp but the producer
            tc::mbar_init(tc::smem_u32(&fb.fin[i]), 1);
            tc::mbar_init(tc::smem_u32(&fb.fin[2 + i]), 1);
        }
        tc::mbar_init(tc::smem_u32(&fb.next), 1);
        tc::mbar_init(tc::smem_u32(&fb.v_part), 1);
        tc::mbar_init(tc::smem_u32(&fb.skew), 1);
        fb.abort = 0;
        tc::fence_barrier_init();
        tc::prefetch_tmap(&qmap);
        tc::prefetch_tmap(&kmap);
        tc::prefetch_tmap(&vmap);
    }
    if (warp == 0) tc::tmem_alloc(tc::smem_u32(&fb.tmem), 512);
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = fb.tmem;
    // the kernel that follows a prefix pass starts on the SMs that this one leaves
    // free, without waiting for it: so the pass's own predecessor must be done first,
    // and the pass hands on, by a release, that it has seen that
    griddep_wait();
    if (a.prefix && blockIdx.x == 0 && threadIdx.x == 0) tc::st_release_gpu(a.ready, a.token);
    griddep_launch_dependents();

    // The next item of a reading warp (all but the producer): its number, then what
    // it is.  False at the end, or when the CTA has been given up.
    auto next_work = [&](int it, Work &w) -> bool {
        if (!wait_all(fb.work_full[it & 1], it >> 1, abort, a.err, PK_WORK)) return false;
        w = fb.work[it & 1];
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(tc::smem_u32(&fb.work_free[it & 1]));
        return !w.end;
    };

    if (warp == 0) {
        // ---------------- items and TMA producer ----------------
        // boxes of a block: `bt` tokens each (a page, or all 128 keys)
        const int bt = a.prefix ? min(KB, 1 << a.kv.page_shift) : KB, nbox = KB / bt;
        const int32_t *table = nullptr;
        if (a.prefix) {
            // any row's table will do: the first token's that is no padding
            int row = -1;
            for (int m0 = 0; m0 < a.M && row < 0; m0 += 32) {
                const int r = m0 + lane < a.M ? load_id(a.trow + m0 + lane) : -1;
                const unsigned ok = __ballot_sync(0xffffffffu, r >= 0 && r < a.kv.rows);
                if (ok) row = __shfl_sync(0xffffffffu, r, __ffs(ok) - 1);
            }
            table = row < 0 ? nullptr : a.kv.table + (size_t)row * a.kv.max_pages;
        }
        bool ok = true, more = true;
        int it = 0, asked = 0, kc = 0, vc = 0, vp = 0, qc0 = 0, qc1 = 0;   // items shown, requests, fills so far
        for (int id = blockIdx.x; ok; ++asked) {
            // ask for the CTA that would start next (its item becomes this CTA's); the
            // answer is read when this item's copies have been issued
            if (lane == 0) {
                tc::mbar_arrive_expect_tx(tc::smem_u32(&fb.next), 16);
                request_next(tc::smem_u32(fb.response), tc::smem_u32(&fb.next));
            }
            __syncwarp();
            const Work w = work_of(a, id);
            if (w.ntok > 0) {
                if (it >= 2) ok = wait_all(fb.work_free[it & 1], (it >> 1) - 1, abort, a.err, PK_WORK);
                if (ok && lane == 0) {
                    fb.work[it & 1] = w;
                    tc::mbar_arrive(tc::smem_u32(&fb.work_full[it & 1]));
                }
                ++it;
            }
            if (w.ntok > 0 && w.nb) {
                // the queries' memory is free only when the last item's scores are through:
                // bring them to L2 meanwhile, and the first K, which has room earlier, in
                if (lane < w.tiles * S::HALVES)
                    prefetch_3d(&qmap, (lane % S::HALVES) * 64, w.h * a.G, w.tok0 + lane / S::HALVES * a.TQ);
                auto load_q = [&]() {
                    for (int i = 0; i < w.tiles && ok; ++i) {
                        int &qc = i ? qc1 : qc0;
                        if (qc) ok = wait_all(fb.q_free[i], qc - 1, abort, a.err, PK_FREE);
                        if (ok && lane == 0) {
                            const uint32_t qb = tc::smem_u32(&fb.q_full[i]);
                            tc::mbar_arrive_expect_tx(qb, (uint32_t)(S::HALVES * a.G * a.TQ * 128));
                            for (int x = 0; x < S::HALVES; ++x)
                                tc::tma_load_3d(tc::smem_u32(sm_q + i * S::TILE + x * BOX), &qmap, x * 64, w.h * a.G, w.tok0 + i * a.TQ, qb);
                        }
                        if (ok) ++qc;
                    }
                };
                for (int f = 0; f < 2 * w.nb && ok; ++f) {   // K_0, the queries, V_0, K_1, ...
                    if (f == 1) load_q();
                    if (!ok) break;
                    const int j = f >> 1, v = f & 1, fill = v ? vc : kc, s = v ? fill % VSLOTS : fill % KSLOTS, turn = v ? fill / VSLOTS : fill / KSLOTS;
                    if (turn) ok = wait_all(v ? fb.v_free[s] : fb.k_free[s], turn - 1, abort, a.err, PK_FREE);
                    if (!ok) break;
                    const int key0 = w.kbeg + j * KB, nv = w.kend - key0;
                    // V of a block that ends inside 16 keys is shown only when the rows behind
                    // its last key are zeroed
                    const bool part = v && j + 1 == w.nb && (nv & 15);
                    const CUtensorMap *map = v ? &vmap : &kmap;
                    const uint32_t bar = tc::smem_u32(part ? &fb.v_part : v ? &fb.v_full[s] : &fb.k_full[s]);
                    unsigned char *tile = (v ? sm_v : sm_k) + s * S::TILE;
                    const uint32_t dst = tc::smem_u32(tile);
                    const int boxes = a.prefix ? min(nbox, (nv + bt - 1) / bt) : 1;
                    if (lane == 0) tc::mbar_arrive_expect_tx(bar, (uint32_t)(boxes * S::HALVES * bt * 128));
                    __syncwarp();
                    if (lane < boxes * S::HALVES) {
                        const int b = lane / S::HALVES, x = lane % S::HALVES;
                        if (a.prefix) {
                            const int key = key0 + b * bt;
                            int page = table ? load_id(table + (key >> a.kv.page_shift)) : -1;
                            if (page < 0 || page >= a.kv.n_pages) {   // reads as zeros (a box outside the tensor)
                                if (table && a.err) atomicExch(a.err, PE_PAGE);
                                page = a.kv.n_pages;
                            }
                            tma_load_4d(dst + x * BOX + b * bt * 128, map, x * 64, key & ((1 << a.kv.page_shift) - 1), w.h, page, bar);
                        } else {
                            tma_load_4d(dst + x * BOX, map, x * 64, w.krow0 + key0, w.h, 0, bar);
                        }
                    }
                    if (v) ++vc;
                    else ++kc;
                    if (part) {
                        ok = wait_all(fb.v_part, vp++, abort, a.err, PK_KV);
                        if (!ok) break;
                        const int words = (16 - (nv & 15)) * 8;
                        for (int y = lane; y < words * S::HALVES; y += 32)
                            *reinterpret_cast<uint4 *>(tile + (y / words) * BOX + nv * 128 + (y % words) * 16) = make_uint4(0, 0, 0, 0);
                        tc::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(tc::smem_u32(&fb.v_full[s]));
                    }
                }
            }
            // the answer; it must be in before the CTA ends, whatever else happened
            const bool in = tc::mbar_wait(tc::smem_u32(&fb.next), asked & 1, a.err, PK_WORK);
            more = __all_sync(0xffffffffu, in) && next_item(tc::smem_u32(fb.response), &id);
            __syncwarp();
            if (!more) break;
        }
        if (ok) {   // show the end
            if (it >= 2) ok = wait_all(fb.work_free[it & 1], (it >> 1) - 1, abort, a.err, PK_WORK);
            if (ok && lane == 0) {
                fb.work[it & 1].end = 1;
                tc::mbar_arrive(tc::smem_u32(&fb.work_full[it & 1]));
            }
        }
        // copies in flight must land before the CTA's shared memory is released
        if (*abort) {
            if (qc0) tc::mbar_wait(tc::smem_u32(&fb.q_full[0]), (qc0 - 1) & 1, nullptr, 0);
            if (qc1) tc::mbar_wait(tc::smem_u32(&fb.q_full[1]), (qc1 - 1) & 1, nullptr, 0);
            for (int f = max(0, kc - KSLOTS); f < kc; ++f) tc::mbar_wait(tc::smem_u32(&fb.k_full[f % KSLOTS]), (f / KSLOTS) & 1, nullptr, 0);
            for (int f = max(0, vc - VSLOTS); f < vc; ++f) tc::mbar_wait(tc::smem_u32(&fb.v_full[f % VSLOTS]), (f / VSLOTS) & 1, nullptr, 0);
            if (vp) tc::mbar_wait(tc::smem_u32(&fb.v_part), (vp - 1) & 1, nullptr, 0);
        }
    } else if (warp == 3 || warp == 12) {
        // ---------------- issuer of tile i's scores (the whole warp waits, one lane issues) ----------------
        // Issuing, committing and waiting take as long as the products themselves: every
        // chain of products has a warp of its own.
        constexpr uint32_t idesc_s = tc::idesc_f16_f32(TM, SB) | Pk<T>::fmt;
        const int i = warp == 3 ? 0 : 1;
        // descriptors differ only in their address field (16-byte units)
        const uint64_t qd = tc::sdesc_k_sw128(tc::smem_u32(sm_q + i * S::TILE)), kd0 = tc::sdesc_k_sw128(tc::smem_u32(sm_k));
        const uint32_t tS = tmem + COL_S + i * 128;
        bool ok = true;
        Work w;
        // blocks of K and scores of this tile so far, items with scores
        for (int it = 0, kc = 0, sc = 0, qc = 0; ok && next_work(it, w); ++it) {
            if (i >= w.tiles || !w.nb) {
                kc += w.nb;
                continue;
            }
            ok = wait_all(fb.q_full[i], qc++, abort, a.err, PK_Q);
            // tile 1 starts when tile 0 is through its first scores, so that the one's
            // softmax meets the other's products from then on
            if (i && !it) ok = ok && wait_all(fb.skew, 0, abort, a.err, PK_P);
            for (int n = 0; n < w.ns && ok; ++n, ++sc) {   // keys 64 n .. 64 n + 63 into buffer sc & 1
                const int half = n & 1, b = sc & 1, kb = kc + (n >> 1), sl = kb % KSLOTS;
                if (!half) ok = wait_all(fb.k_full[sl], kb / KSLOTS, abort, a.err, PK_KV);
                // the scores lie over P of two blocks ago: the product that reads it comes first
                if (sc >= 2) ok = ok && wait_all(fb.pv_done[i][b], (sc >> 1) - 1, abort, a.err, PK_PV);
                if (!ok) break;
                tc::fence_after_sync();
                const uint64_t kd = kd0 + (uint32_t)(sl * (S::TILE >> 4) + half * (SB * 128 >> 4));
                const uint32_t d = tS + b * SB;
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t off = (uint32_t)(((kk >> 2) * BOX + (kk & 3) * 32) >> 4);
                        tc::mma_ss_f16(d, qd + off, kd + off, idesc_s, kk ? 1u : 0u);
                    }
                    tc::mma_commit(tc::smem_u32(&fb.s_full[i][b]));
                    if (half || n + 1 == w.ns) {
                        tc::mma_commit(tc::smem_u32(&fb.k_free[sl]));
                        if (w.tiles == 1) tc::mma_commit(tc::smem_u32(&fb.k_free[sl]));   // for the tile that is not there
                    }
                    if (n + 1 == w.ns) tc::mma_commit(tc::smem_u32(&fb.q_free[i]));
                }
                __syncwarp();
            }
            kc += w.nb;
        }
        // everything issued must finish before TMEM is freed
        if (elect_one()) tc::mma_commit(tc::smem_u32(&fb.fin[2 + i]));
        __syncwarp();
        tc::mbar_wait(tc::smem_u32(&fb.fin[2 + i]), 0, nullptr, 0);
    } else if (warp == 1 || warp == 2) {
        // ---------------- issuer of tile i's O += P V ----------------
        constexpr uint32_t idesc_pv = tc::idesc_f16_f32(TM, D) | (1u << 16) | Pk<T>::fmt;   // B (V) MN-major
        const int i = warp - 1;
        const uint64_t vd0 = tc::sdesc_mn_sw128(tc::smem_u32(sm_v), BOX);
        const uint32_t tS = tmem + COL_S + i * 128, tO = tmem + COL_O + i * 128;
        bool ok = true;
        Work w;
        for (int it = 0, vc = 0, sc = 0, oc = 0; ok && next_work(it, w); ++it) {
            if (i >= w.tiles || !w.nb) {
                vc += w.nb;
                continue;
            }
            if (oc) ok = wait_all(fb.o_free[i], oc - 1, abort, a.err, PK_PV);   // the last item's O has been read
            ++oc;
            for (int n = 0; n < w.ns && ok; ++n, ++sc) {
                const int half = n & 1, b = sc & 1, vb = vc + (n >> 1), sl = vb % VSLOTS;
                const uint64_t vd = vd0 + (uint32_t)(sl * (S::TILE >> 4) + half * (SB * 128 >> 4));
                const int nv = n + 1 < w.ns ? SB : w.kend - w.kbeg - n * SB, ks = (nv + 15) / 16;   // 16-key steps that hold keys
                if (!half) ok = wait_all(fb.v_full[sl], vb / VSLOTS, abort, a.err, PK_KV);
                ok = ok && wait_all(fb.p_full[i][b], sc >> 1, abort, a.err, PK_P);
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
                    if (half || n + 1 == w.ns) {
                        tc::mma_commit(tc::smem_u32(&fb.v_free[sl]));
                        if (w.tiles == 1) tc::mma_commit(tc::smem_u32(&fb.v_free[sl]));
                    }
                }
                __syncwarp();
            }
            vc += w.nb;
        }
        if (elect_one()) tc::mma_commit(tc::smem_u32(&fb.fin[i]));
        __syncwarp();
        tc::mbar_wait(tc::smem_u32(&fb.fin[i]), 0, nullptr, 0);
    } else {
        // ---------------- softmax and epilogue: thread = query row ----------------
        const int i = (warp - 4) >> 2, quarter = warp & 3;
        const int r = quarter * 32 + lane, j0 = r / a.G, gh = r - j0 * a.G;   // row of the tile, its token and head
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const uint32_t tS = tmem + lane_base + COL_S + i * 128, tO = tmem + lane_base + COL_O + i * 128;
        const uint64_t sc2 = pack2(a.scale_log2, a.scale_log2);
        const bool wide = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
        const int tk = i * a.TQ + j0;                              // token of the item
        for (int it = 0, sc = 0;; ++it) {
            // the item's description stays where it is until the end: registers are
            // what this warp is short of
            if (!wait_all(fb.work_full[it & 1], it >> 1, abort, a.err, PK_WORK)) break;
            const Work &w = fb.work[it & 1];
            if (w.end) break;
            if (i >= w.tiles) {
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(tc::smem_u32(&fb.work_free[it & 1]));
                continue;
            }
            const bool valid = r < a.G * a.TQ && tk < w.ntok;
            int lim = -1;                                          // last key the row sees
            bool pad = !valid;
            if (valid) {
                if (!a.prefix) lim = a.causal ? min(w.first_lim + tk, w.kend - 1) : w.kend - 1;
                else {
                    const int row = load_id(a.trow + w.tok0 + tk), pos = load_id(a.tpos + w.tok0 + tk);
                    pad = row < 0;
                    if (row < a.kv.rows) lim = min(pos, w.kend - 1);   // a row outside the table sees nothing
                }
            }
            lim = pad ? 0x3fffffff : lim - w.kbeg;   // rows nobody reads need no mask
            const int ns = w.ns;
            float m_used = -INFINITY, l = 0.f;
            bool ok = true;
            for (int n = 0; n < ns; ++n, ++sc) {
                const int b = sc & 1;
                ok = wait_all(fb.s_full[i][b], sc >> 1, abort, a.err, PK_S);
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
                    ok = wait_all(fb.pv_done[i][b ^ 1], (sc - 1) >> 1, abort, a.err, PK_PV);
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
                    const uint64_t e = exp2_2(z);
                    sum2[x & 1] = add2(sum2[x & 1], e);
                    p[x] = Pk<T>::pack(lo2(e), hi2(e));
                }
                tc::tmem_st32(tS + b * SB, p);
                tc::tmem_wait_st();
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(tc::smem_u32(&fb.p_full[i][b]));
                if (n == 0 && it == 0 && warp == 4 && lane == 0) tc::mbar_arrive(tc::smem_u32(&fb.skew));
                sum2[0] = add2(sum2[0], sum2[1]);
                l = l * alpha + (lo2(sum2[0]) + hi2(sum2[0]));
            }
            if (ok && ns) {
                ok = wait_all(fb.pv_done[i][(sc - 1) & 1], (sc - 1) >> 1, abort, a.err, PK_PV);
                ok = __all_sync(0xffffffffu, ok && !*abort);
                tc::fence_after_sync();
            }
            if (!ok) break;
            const float inv = l != 0.f ? 1.f / l : 0.f;
            T *dst = reinterpret_cast<T *>(a.out) + ((size_t)(w.tok0 + tk) * a.Hq + w.h * a.G + gh) * D;
            const size_t part_rows = (size_t)a.M * a.G, part_row = (size_t)(w.tok0 + tk) * a.G + gh;
            const size_t part = (size_t)w.split * a.Hkv + w.h;
            // behind this arrival the producer may write the item after next into w: nothing
            // reads w below
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(tc::smem_u32(&fb.work_free[it & 1]));
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t acc[32];
                __syncwarp();
                if (ns) {
                    tc::tmem_ld32(tO + c * 32, acc);
                    tc::tmem_wait_ld();
                }
                if (ns && c + 1 == D / 32) {   // O may be written again
                    tc::fence_before_sync();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(tc::smem_u32(&fb.o_free[i]));
                }
                const bool live = ns && l != 0.f;
#pragma unroll
                for (int x = 0; x < 32; ++x)
                    if (!live) acc[x] = 0u;
                if (!pad && a.prefix) {
                    // [split][KV head][8 features][row][8]: a warp's 32 rows are one kilobyte
                    float *p = a.o_part + (part * (D / 8) + c * 4) * part_rows * 8 + part_row * 8;
#pragma unroll
                    for (int x = 0; x < 4; ++x) store32(p + x * part_rows * 8, acc + x * 8);
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
            if (a.prefix && !pad)
                *reinterpret_cast<float2 *>(a.ml_part + (part * part_rows + part_row) * 2) = make_float2(m_used, l);
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 0) {
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

int prefix_items(int M, int n_heads, int n_kv) {
    const int TQ = TM / (n_heads / n_kv);
    return (int)std::min<int64_t>((int64_t)((M + 2 * TQ - 1) / (2 * TQ)) * n_kv, 0x7fffffff);
}

int prefix_splits(int M, int n_heads, int n_kv, int prefix_len, int sm_count) {
    const int64_t items = prefix_items(M, n_heads, n_kv), blocks = (prefix_len + KB - 1) / KB;
    // one wave of CTAs, two key blocks each at least; half a wave when a whole one
    // would have few blocks each: start and end of a CTA then count for more than
    // its blocks, and the rows' own keys are read on the other SMs meanwhile (64
    // tokens over 8,192 shared keys and up to 512 own ones: 46.7 us on all, 44.5 on a
    // third, 41.3 on half).  The host does not know the rows' own keys, and long ones
    // behind a short prefix are better off without a pass: 64 rows of 32 / 8 heads over
    // 2,048 shared keys took, read once against row by row, 39 and 69 us with 256 own
    // keys, 77 and 93 with 1,024, 217 and 176 with 4,096, 810 and 688 with 16,384.
    int64_t sms = sm_count;
    if (blocks * items < FEW_BLOCKS * sms) sms /= 2;
    return (int)std::max<int64_t>(1, std::min<int64_t>(sms / items, (blocks + 1) / 2));
}

int prefix_max_splits(int M, int n_heads, int n_kv, int prefix_len, int sm_count) {
    const int64_t items = prefix_items(M, n_heads, n_kv), blocks = (prefix_len + KB - 1) / KB;
    return (int)std::max<int64_t>(1, std::min<int64_t>(sm_count / items, (blocks + 1) / 2));
}

cudaError_t prefix_attn(const PagedKV &kv, const PagedQuery &q, int prefix_len, const PrefixPartials &part, cudaStream_t st) {
    Args a = {};
    a.prefix = 1; a.kv = kv; a.trow = q.trow; a.tpos = q.tpos; a.M = q.M; a.prefix_len = prefix_len; a.splits = part.splits;
    a.o_part = part.o; a.ml_part = part.ml; a.ready = part.ready; a.token = part.token;
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
