// Attention of many query rows over spans of an fp16 cache on the 5th-generation tensor cores (head_dim 64 and 128): the chunks of a
// prompt under a window, and a large batch's rows over a shared prefix.  attn_span.cu has the rest, and joins partial results.
//
// What bounds it: 128 rows x 64 keys take 768 clocks of the tensor pipe at head_dim 128 (S, and P V twice), and their 8192 exponentials 512 clocks of
// the SM's sixteen a clock; neither is reached in a short call (66 % of the tensor pipe), since scores, exponentials and P V of a row wait for one another.  So an SM has two
// CTAs, and a CTA two tiles of scores: while the softmax has one, the tensor pipe has the other one's products and the other CTA's.  In calls one
// after another for a second the 1000 W limit is the bound.
//
// * Q (128 rows), K and V tiles of 64 keys in shared memory, 128-byte swizzle, K and V in two stages by TMA.  Tiles that are not 64 rows
//   in one piece (the first rows, the end of a sequence) come in by cp.async, places past the last key zero-filled: what a cache holds there
//   is nobody's business.  K is a K-major operand, V an MN-major one, so neither is transposed.
// * Two buffers of scores and the output accumulators in tensor memory, half of it a CTA.  A thread has a row's 64 scores; P, as two
//   fp16 halves (22 bits of a weight, as in the framework's other attention), overwrites them, 32 keys at a time: the high halves take the first 32
//   columns, the low ones the others, and both are read from there as A operands.
// * Which tiles every row of a warp sees is worked out once, not per tile (2048 tokens behind 6000 under a window of 4096, 32/8 heads, head_dim
//   128: 172 -> 162 us).
// * The output is rescaled only when a row's maximum grows by more than 2^8; the stale maximum cancels in the normalisation.
// Two CTAs of 128 rows, a thread a row, two buffers of 64 scores; measured while P was one half: 136 us for the kernel of that call, where one CTA an
// SM of 256 rows took 147 to 155, and four warps for the even tiles of keys and four for the odd ones 163.  With both halves of P the call takes 183 us
// cold (152 with one half; 750 TFLOP/s of the operations that the rows ask for), 64 sequences of 64/8 heads over a prefix of 32768 with own keys and join
// 141 (124); at head_dim 64 160 and 113.  P in pieces of 16 keys on its way to tensor memory keeps the softmax within 128 registers (head_dim 64,
// the first call: 164 -> 160 us).
// Every wait is bounded: on a time-out the sticky error word is set, tensor memory is freed and the CTA returns.
#include <cuda.h>

#include "attn_span.cuh"

namespace alloyb {
namespace st5 {

using sp::Params;
using sp::Seq;

constexpr int ROWS = 128, KT = 64, STAGES = 2, AHEAD = 3;
constexpr int THREADS = 8 * 32;              // warps 0 and 3 copy K and V, 1 issues the MMAs, 4-7 are the softmax
constexpr int Q_HALF = ROWS * 128, KV_HALF = KT * 128;       // bytes of a tile's rows x 64 halves
constexpr uint32_t SPIN = 1u << 22;

static __device__ int g_tc_error = 0;        // sticky: a bounded wait of this file's kernel ran out

template <int D>
struct Cfg {
    static constexpr int Q = D / 64 * Q_HALF, TILE = D / 64 * KV_HALF;
    static constexpr int SMEM = 1024 + Q + 2 * STAGES * TILE + 256;
    static constexpr int COLS = 256;         // tensor-memory columns: two buffers of 64 scores, D of outputs; two CTAs an SM have all of it
};
struct alignas(64) Args {
    CUtensorMap k, v;                        // (D, rows, heads), boxes of 64 elements x KT rows, 128-byte swizzle
    Params p;
};
struct Bars {
    uint64_t k_full[STAGES], v_full[STAGES], k_empty[STAGES], v_empty[STAGES];
    uint64_t s_full[2], p_half[2], p_full[2];        // [buffer]
    uint32_t tmem_base;
};

using sp::ex2;
using sp::pack_h2;
using sp::s32;

__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t n) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(s32(b)), "r"(n)); }
__device__ __forceinline__ void bar_arrive(uint64_t* b) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(s32(b)) : "memory"); }
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(s32(b)), "r"(parity)
                 : "memory");
    return ok != 0;
}
__device__ __noinline__ bool bar_wait_slow(uint64_t* b, uint32_t parity) {
    for (uint32_t i = 0; i < SPIN; ++i) {
        if (bar_try(b, parity)) return true;
        if (i > 32) __nanosleep(64);
    }
    atomicExch(&g_tc_error, 1);
    return false;
}
__device__ __forceinline__ void bar_wait(bool& ok, uint64_t* b, uint32_t parity) {
    if (ok && !bar_try(b, parity)) ok = bar_wait_slow(b, parity);
}
// Shared-memory operand in the 128-byte swizzle, rows of 128 bytes, groups of eight rows 1024 bytes apart.  K-major: the leading offset is
// unused; MN-major: it leads to the next 64 elements.
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t leading) {
    return static_cast<uint64_t>((addr >> 4) & 0x3fffu) | static_cast<uint64_t>((leading >> 4) & 0x3fffu) << 16 |
           static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
// kind::f16, fp16 operands, fp32 accumulators, M = 128; b_mn: B is MN-major
__device__ __forceinline__ constexpr uint32_t umma_idesc(int n, bool b_mn) {
    return 1u << 4 | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n) >> 3) << 17 | (128u >> 4) << 24;
}
// A warp's issue, all lanes in step: `lead` is 1 in the lane that does it.
__device__ __forceinline__ uint32_t elect() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(accumulate), "r"(lead)
                 : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate, uint32_t lead) {
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
                 "r"(idesc), "r"(accumulate), "r"(lead)
                 : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* b, uint32_t lead) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(s32(b)), "r"(lead)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
    uint32_t* u = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
          "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]),
          "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]),
          "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
    uint32_t* u = reinterpret_cast<uint32_t*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
                   "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr), "r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
        "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Two fp32 values in one 64-bit register and the two-wide instructions on them.
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unf2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(s32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(map),
                 "r"(s32(bar)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* map, int x, int y, int z) {
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global [%0, {%1, %2, %3}];" ::"l"(map), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Byte offset of 16-byte piece c of a row in a tile: halves of 64 elements (`half` bytes), each in the 128-byte swizzle.
__device__ __forceinline__ uint32_t piece_at(int row, int c, int half) { return (c >> 3) * half + row * 128 + (((c & 7) ^ (row & 7)) << 4); }

// Grid (tiles * splits, KV_H, B); PREFIX: rows of the whole batch over the shared prefix, grid z 1, partial results only.
template <int D, bool PREFIX>
__global__ void __launch_bounds__(THREADS, 2) span_tc_kernel(const __grid_constant__ Args A) {
    const Params& P = A.p;
    using C = Cfg<D>;
    constexpr int TILE = C::TILE, PIECES = D / 8;
    extern __shared__ uint8_t smem_raw[];
    __shared__ float back[ROWS];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t q_s = s32(smem), k_s = q_s + C::Q, v_s = k_s + STAGES * TILE;
    Bars* bars = reinterpret_cast<Bars*>(smem + C::Q + 2 * STAGES * TILE);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int splits = PREFIX ? P.pre_splits : P.splits, tiles = gridDim.x / splits;
    const int split = blockIdx.x % splits, tile = tiles - 1 - blockIdx.x / splits;      // the rows with the most keys go first
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int rows = P.n * P.G, all_rows = PREFIX ? rows * P.B : rows, row0 = tile * ROWS;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            bar_init(&bars->k_full[s], 1);
            bar_init(&bars->v_full[s], 1);
            bar_init(&bars->k_empty[s], 1);
            bar_init(&bars->v_empty[s], 1);
        }
        for (int h = 0; h < 2; ++h) {
            bar_init(&bars->s_full[h], 1);
            bar_init(&bars->p_half[h], 4);
            bar_init(&bars->p_full[h], 4);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // Tensor memory behind the wait, and what follows may begin only once every CTA has its own: a CTA of the launch before or behind that
    // shares the SM could otherwise wait for the columns that this one holds while this one waits for it.
    pdl_wait();
    if (PREFIX && threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) sp::tell_begun(P);
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s32(&bars->tmem_base)), "r"(C::COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    const int tok0 = row0 / P.G, tok1 = min(P.n, (row0 + ROWS - 1) / P.G + 1);
    Seq sq = {0, 0, 0, P.P};
    if (!PREFIX) sq = sp::seq_at(P, sp::live_pos(P, b, tile == 0 && kvh == 0 && split == 0 && threadIdx.x == 0), tok0, tok1);
    const int steps = (sq.keys + KT - 1) / KT, per = (steps + splits - 1) / splits;
    const int step0 = min(steps, split * per), n_tiles = min(steps, step0 + per) - step0;
    const int64_t head = PREFIX ? kvh * P.p_hs : (static_cast<int64_t>(b) * P.KV_H + kvh) * P.S * D;

    // ---- Q rows; dead rows are zero
    constexpr int WARPS = THREADS / 32, BATCH = 8;
    for (int i0 = 0; i0 * WARPS < ROWS; i0 += BATCH) {
        sp::QRow<D> qr[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int r = warp + (i0 + i) * WARPS, R = row0 + r, rb = PREFIX ? R / rows : b, rest = PREFIX ? R - rb * rows : R, tok = rest / P.G, hg = rest - tok * P.G;
            qr[i].read(P.q, rb * P.q_bs + (kvh * P.G + hg) * P.q_hs + tok * P.q_ts, P.q_vec != 0, R < all_rows, lane);
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int r = warp + (i0 + i) * WARPS;
            const float f = qr[i].put([&](int d) { return q_s + piece_at(r, d >> 3, Q_HALF) + (d & 7) * 2; }, P.q_dtype, lane);
            if (lane == 0) back[r] = f * P.scale_log2;
        }
    }
    fence_async();
    fence_before();
    __syncthreads();
    fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = bars->tmem_base;
    bool ok = true;

    if (warp < 4) {
        if (warp == 1) {
            // ------------------------------------------------ MMA issue
            const uint32_t lead = elect();
            const uint64_t q_desc = umma_desc(q_s, 16), k_desc = umma_desc(k_s, 16), v_desc = umma_desc(v_s, KV_HALF);
            auto scores = [&](int j, int h) {                                 // of tile j, into buffer h
                const int s = j % STAGES;
                bar_wait(ok, &bars->k_full[s], (j / STAGES) & 1);
                fence_after();
                if (!ok) return;
                const uint64_t kd = k_desc + ((s * TILE) >> 4);
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    umma_ss(tmem + h * KT, q_desc + (((kk >> 2) * Q_HALF + (kk & 3) * 32) >> 4), kd + (((kk >> 2) * KV_HALF + (kk & 3) * 32) >> 4),
                            umma_idesc(KT, false), kk > 0, lead);
                umma_commit(&bars->s_full[h], lead);
                umma_commit(&bars->k_empty[s], lead);
            };
            if (n_tiles > 0) scores(0, 0);
            if (n_tiles > 1) scores(1, 1);
            for (int j0 = 0; j0 < n_tiles && ok; j0 += 2) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int j = j0 + h, s = j % STAGES;
                    if (j >= n_tiles) break;
                    bar_wait(ok, &bars->v_full[s], (j / STAGES) & 1);
#pragma unroll
                    for (int kk = 0; kk < KT / 16; ++kk) {
                        if (kk == 0 || kk == KT / 32) {                       // P comes in two pieces
                            bar_wait(ok, kk == 0 ? &bars->p_half[h] : &bars->p_full[h], (j >> 1) & 1);
                            fence_after();
                            if (!ok) break;
                        }
                        const uint64_t vd = v_desc + ((s * TILE + kk * 2048) >> 4);
                        umma_ts(tmem + 2 * KT, tmem + h * KT + kk * 8, vd, umma_idesc(D, true), j > 0 || kk > 0, lead);
                        umma_ts(tmem + 2 * KT, tmem + h * KT + KT / 2 + kk * 8, vd, umma_idesc(D, true), 1, lead);
                    }
                    if (!ok) break;
                    umma_commit(&bars->v_empty[s], lead);
                    // behind P V, in the order of issue: S may take P's place, and whoever sees it complete has that P V too
                    if (j + 2 < n_tiles) scores(j + 2, h);
                    else umma_commit(&bars->s_full[h], lead);
                }
            }
            __syncwarp();
        } else if (warp == 0 || warp == 3) {
            // ------------------------------------------------ tiles of K (warp 0) and V (warp 3)
            const bool is_v = warp == 3;
            const int c = lane % PIECES, r0 = lane / PIECES;
            const int z = PREFIX ? kvh : b * P.KV_H + kvh;
            const __half* src = PREFIX ? nullptr : (is_v ? P.v : P.k) + head + c * 8;
            // Two stages of shared memory hide the way from L2; tiles on their way into L2 need none
            auto ahead = [&](int j) {
                const int place0 = (step0 + j) * KT;
                if (lane == 0 && j < n_tiles && (PREFIX || (place0 >= sq.sink && place0 + KT <= sq.keys))) {
#pragma unroll
                    for (int h = 0; h < D / 64; ++h) tma_prefetch_3d(is_v ? &A.v : &A.k, h * 64, PREFIX ? place0 : sq.row_of(place0), z);
                }
            };
            for (int j = STAGES; j < AHEAD; ++j) ahead(j);
            for (int j = 0; j < n_tiles; ++j) {
                const int s = j % STAGES;
                ahead(j + AHEAD);
                uint64_t* full = is_v ? &bars->v_full[s] : &bars->k_full[s];
                if (j >= STAGES) bar_wait(ok, is_v ? &bars->v_empty[s] : &bars->k_empty[s], ((j / STAGES) - 1) & 1);
                const uint32_t dst = (is_v ? v_s : k_s) + s * TILE;
                const int place0 = (step0 + j) * KT;
                // (rows past the prefix's last are outside the map: TMA fills them with zeros)
                if (PREFIX || (place0 >= sq.sink && place0 + KT <= sq.keys)) {
                    if (lane == 0 && ok) {
                        bar_expect(full, TILE);
#pragma unroll
                        for (int h = 0; h < D / 64; ++h) tma_3d(dst + h * KV_HALF, is_v ? &A.v : &A.k, h * 64, PREFIX ? place0 : sq.row_of(place0), z, full);
                    }
                } else {
                    if (ok) {
#pragma unroll 8
                        for (int i = 0; i < KT * PIECES / 32; ++i) {
                            const int r = r0 + i * (32 / PIECES);
                            const bool live = place0 + r < sq.keys;
                            sp::copy16(dst + piece_at(r, c, KV_HALF), src + static_cast<int64_t>(live ? sq.row_of(place0 + r) : 0) * D, live);
                        }
                    }
                    sp::copy_commit();
                    sp::copy_wait<0>();
                    fence_async();                                    // to the tensor pipe's proxy
                    __syncwarp();
                    if (lane == 0) bar_arrive(full);
                }
            }
        }
    } else {
        // ------------------------------------------------ softmax, a thread a row
        const int r = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const int R = row0 + r, pos = sq.pos + R / P.G;                       // (of a chunk) last row of the cache that this one may see
        const float scale = back[r];
        // tiles whole0 .. whole1 - 1 of the sequence are seen by all rows of the warp: no key behind the earliest row, none before the latest
        // row's window
        int whole0 = 0, whole1 = sq.keys / KT;
        if (!PREFIX) {
            const int first = sq.pos + (R - lane) / P.G, last = sq.pos + (R - lane + 31) / P.G;
            whole1 = min(whole1, (first + 1 - sq.lo + sq.sink) / KT);
            if (P.window > 0) whole0 = max((sq.sink + KT - 1) / KT, (last - P.window + 1 - sq.lo + sq.sink + KT - 1) / KT);
        }
        float m_run = -INFINITY, l_run = 0.f;                                 // (l: times 64 like the accumulators)
        for (int j = 0; j < n_tiles; ++j) {
            const uint32_t buf = lanes + (j & 1) * KT;
            bar_wait(ok, &bars->s_full[j & 1], (j >> 1) & 1);
            fence_after();
            float s[KT];
#pragma unroll
            for (int c = 0; c < KT / 32; ++c) tmem_ld32(buf + c * 32, *reinterpret_cast<float(*)[32]>(s + c * 32));
            wait_ld();
            if (step0 + j < whole0 || step0 + j >= whole1) {
                // place e of this tile is seen if e <= hi and (e > lo or e < sk): as bits, 32 places a word
                const int at = (step0 + j) * KT, hi = min(sq.keys - 1, PREFIX ? sq.keys - 1 : pos - sq.lo + sq.sink) - at;
                const int lo = PREFIX || P.window <= 0 ? -1 : pos - P.window - sq.lo + sq.sink - at, sk = PREFIX ? 0 : P.sinks - at;
#pragma unroll
                for (int c = 0; c < KT / 32; ++c) {
                    const uint32_t seen = sp::bits_below(hi + 1 - 32 * c) & (~sp::bits_below(lo + 1 - 32 * c) | sp::bits_below(sk - 32 * c));
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (!(seen >> e & 1u)) s[c * 32 + e] = -INFINITY;
                }
            }
            float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < KT; e += 8)
#pragma unroll
                for (int k = 0; k < 4; ++k) mx4[k] = max3(mx4[k], s[e + k], s[e + 4 + k]);
            const float mx = fmaxf(max3(mx4[0], mx4[1], mx4[2]), mx4[3]) * scale;
            const bool grow = mx > m_run + sp::RESCALE_LOG2;
            if (__any_sync(0xffffffffu, grow)) {
                const float alpha = grow ? ex2(m_run - mx) : 1.0f;
                if (grow) m_run = mx;
                l_run *= alpha;
                if (j > 0) {
                    bar_wait(ok, &bars->s_full[(j & 1) ^ 1], (((j - 1) >> 1) + 1) & 1);       // behind the last P V
                    fence_after();
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        float o[16];
                        uint32_t w[16];
                        const uint32_t at = lanes + 2 * KT + c * 16;
                        tmem_ld16(at, o);
                        wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(o[e] * alpha);
                        tmem_st16(at, w);
                    }
                    wait_st();
                }
            }
            const float sub = m_run == -INFINITY ? 0.f : sp::P_BIAS_LOG2 - m_run;
            const uint64_t scale2 = f2(scale, scale), sub2 = f2(sub, sub);
            uint64_t sum[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
            for (int c = 0; c < KT / 16; ++c) {
                uint32_t p[8], low[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float x0, x1;
                    unf2(f2_fma(f2(s[c * 16 + 2 * e], s[c * 16 + 2 * e + 1]), scale2, sub2), x0, x1);
                    x0 = ex2(x0);
                    x1 = ex2(x1);
                    sum[e & 1] = f2_add(sum[e & 1], f2(x0, x1));
                    p[e] = pack_h2(x0, x1);
                    const float2 high = __half22float2(*reinterpret_cast<const __half2*>(&p[e]));
                    low[e] = pack_h2(x0 - high.x, x1 - high.y);
                }
                tmem_st8(buf + c * 8, p);
                tmem_st8(buf + KT / 2 + c * 8, low);
                if (c % 2 == 1) {                                             // 32 keys at a time
                    wait_st();
                    fence_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(c == 1 ? &bars->p_half[j & 1] : &bars->p_full[j & 1]);
                }
            }
            float a0, a1, b0, b1;
            unf2(sum[0], a0, a1);
            unf2(sum[1], b0, b1);
            l_run += (a0 + a1) + (b0 + b1);
        }
        // ---- normalise and store
        if (n_tiles > 0) {
            bar_wait(ok, &bars->s_full[(n_tiles - 1) & 1], (((n_tiles - 1) >> 1) + 1) & 1);
            fence_after();
        }
        const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
        const bool row_live = ok && R < all_rows, direct = !PREFIX && splits == 1 && P.pre_o == nullptr;
        const int tok = R / P.G, hg = R - tok * P.G;
        const int64_t slot = ((static_cast<int64_t>(PREFIX ? 0 : b) * P.KV_H + kvh) * tiles + tile) * splits + split;
        if (row_live && !direct)
            (PREFIX ? P.pre_lse : P.part_lse)[slot * ROWS + r] = l_run == 0.f ? -INFINITY : m_run + log2f(l_run) - sp::P_BIAS_LOG2;
        float* po = (PREFIX ? P.pre_o : P.part_o) + (slot * ROWS + r) * D;
        const int64_t at = ((static_cast<int64_t>(b) * P.n_all + tok) * P.H + kvh * P.G + hg) * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
            float o[32];
            if (n_tiles > 0) {
                tmem_ld32(lanes + 2 * KT + c * 32, o);
                wait_ld();
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0.f;
            }
            if (row_live) {
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const float4 x = make_float4(o[4 * q] * inv, o[4 * q + 1] * inv, o[4 * q + 2] * inv, o[4 * q + 3] * inv);
                    if (direct) sp::store4(P.out, P.q_dtype, at + c * 32 + q * 4, x.x, x.y, x.z, x.w);
                    else *reinterpret_cast<float4*>(po + c * 32 + q * 4) = x;
                }
            }
        }
    }
    if (!ok)
        for (uint32_t i = 0; i < 1024; ++i) __nanosleep(512);                 // a wait ran out: let copies and products in flight end
    fence_before();
    __syncthreads();
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::COLS));
}

// The new tokens' rows into the cache, ahead of a kernel that reads them there.
template <int D>
__global__ void __launch_bounds__(256) span_append_kernel(const Params P) {
    pdl_launch_dependents();
    constexpr int PIECES = D / 8;
    const int tok = blockIdx.x * (256 / PIECES) + threadIdx.x / PIECES, c = threadIdx.x % PIECES * 8, kvh = blockIdx.y, b = blockIdx.z;
    pdl_wait();
    if (tok >= P.n) return;
    const int pos = sp::live_pos(P, b, false);
    if (pos < 0) return;
    const int64_t from = b * P.n_bs + kvh * P.n_hs + tok * P.n_ts + c, to = ((static_cast<int64_t>(b) * P.KV_H + kvh) * P.S + pos + tok) * D + c;
    *reinterpret_cast<uint4*>(P.k + to) = ld_after_wait(P.nk + from);
    *reinterpret_cast<uint4*>(P.v + to) = ld_after_wait(P.nv + from);
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode_fn() {
    static EncodeFn fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult qr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qr) != cudaSuccess || qr != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}
static bool map_rows(CUtensorMap* m, const __half* base, int D, int64_t rows, int64_t heads, int64_t head_stride) {
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(heads)};
    const cuuint64_t pitch[2] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(head_stride) * 2};
    const cuuint32_t box[3] = {64, KT, 1}, step[3] = {1, 1, 1};
    return encode_fn()(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), dims, pitch, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool PREFIX>
static int launch(dim3 grid, cudaStream_t st, const Params& P) {
    auto kern = span_tc_kernel<D, PREFIX>;
    static bool ready[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
    cudaError_t e = encode_fn() ? cudaSuccess : cudaErrorNotSupported;
    if (e == cudaSuccess && !ready[dev]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM);
        if (e == cudaSuccess) ready[dev] = true;
    }
    Args a;
    a.p = P;
    if (e == cudaSuccess) {
        const int64_t rows = PREFIX ? P.P : P.S, heads = PREFIX ? P.KV_H : static_cast<int64_t>(P.B) * P.KV_H, apart = PREFIX && P.KV_H > 1 ? P.p_hs : rows * D;
        auto map = [&] { return map_rows(&a.k, PREFIX ? P.pk : P.k, D, rows, heads, apart) && map_rows(&a.v, PREFIX ? P.pv : P.v, D, rows, heads, apart); };
        // (a host thread's first call of the driver may find no current context, which cudaSetDevice gives it)
        if (!map() && ((e = cudaSetDevice(dev)) != cudaSuccess || !map())) e = e != cudaSuccess ? e : cudaErrorInvalidValue;
    }
    if (e == cudaSuccess && !PREFIX && P.nk) e = launch_pdl(span_append_kernel<D>, dim3((P.n + 2048 / D - 1) / (2048 / D), P.KV_H, P.B), dim3(256), 0, st, P);
    if (e == cudaSuccess) e = launch_pdl(kern, grid, dim3(THREADS), Cfg<D>::SMEM, st, a);
    if (e != cudaSuccess) {
        set_cuda_error(e);
        return ALLOYB_E_CUDA;
    }
    return ALLOYB_OK;
}

}  // namespace st5

// Launches of span_tc_kernel for attn_span.cu, which has checked the sizes (D 64 or 128) and laid the workspace out.
int launch_span_tc(const sp::Params& P, int D, bool prefix, dim3 grid, cudaStream_t st) {
    if (D == 64) return prefix ? st5::launch<64, true>(grid, st, P) : st5::launch<64, false>(grid, st, P);
    return prefix ? st5::launch<128, true>(grid, st, P) : st5::launch<128, false>(grid, st, P);
}

cudaError_t span_tc_status(int* status, int clear) {
    cudaError_t e = cudaMemcpyFromSymbol(status, sp::g_span_status, sizeof(int));
    if (e == cudaSuccess && clear && *status) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(sp::g_span_status, &zero, sizeof(int));
    }
    return e;
}

int span_tc_device_error(int clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, st5::g_tc_error, sizeof(int)) != cudaSuccess) return 0;
    if (clear && v) {
        const int z = 0;
        cudaMemcpyToSymbol(st5::g_tc_error, &z, sizeof(int));
    }
    return v;
}

}  // namespace alloyb
