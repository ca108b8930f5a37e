// Pieces shared by the kernels of attn_span.cu: attention of a few query tokens over spans of an fp16 cache.
#pragma once
#include "common.cuh"

namespace alloyb {
namespace sp {

constexpr float P_BIAS_LOG2 = 6.0f;      // probabilities enter P * V times 64: fp16 keeps 11 bits of one down to 2^-20 of the row's largest
constexpr float RESCALE_LOG2 = 8.0f;     // accumulators follow a row's maximum in steps of this (P then stays below 2^14)
constexpr int MAX_BATCH = 1024;          // sequences per call: every warp of the stream kernel walks all their positions, 32 a round and twice, before it begins
constexpr int STEP = 64;                 // keys that a CTA takes at a time
constexpr int WARPS = 4;

// Sticky word that alloyb_span_status reads, and its bit.
enum { SPAN_POS_RANGE = 1 };
static __device__ int g_span_status = 0;

// Rows of one call: row R of a (sequence, KV head) is token R / G, head R % G of the group.
struct Params {
    const void* q;
    int64_t q_bs, q_hs, q_ts;            // strides in elements: sequence, head, token
    int q_dtype;
    int q_vec;                           // rows may be read 16 bytes at a time
    __half *k, *v;                       // (B, KV_H, S, D)
    int S;
    const __half *nk, *nv;               // the new tokens' rows; null: the cache holds them already
    int64_t n_bs, n_hs, n_ts;
    const int32_t* pos;
    int pos_count;
    void* out;                           // (B, n_all, H, D)
    int B, H, KV_H, G, n;
    int n_all, tok0;                     // the call's tokens, of which these launches have n from tok0 on (q, nk and out begin at tok0)
    int window, sinks;                   // window 0: every position up to the row's own
    float scale_log2;
    const __half *pk, *pv;               // shared prefix (KV_H, P, D)
    int64_t p_hs;
    int P;
    float* part_o;                       // [slot][row][D], normalised
    float* part_lse;                     // [slot][row], log2
    int* cum;                            // B + 1: steps of the sequences before (written by the stream kernel for the merge)
    int ctas;                            // of the stream kernel
    int splits, tiles, tile_rows;        // of the row-tile kernels: CTAs per tile, tiles per (sequence, KV head), rows of a tile
    float* pre_o;                        // the prefix's partials, [KV head][tile][split][row][D]
    float* pre_lse;
    int pre_splits, pre_tile_rows;
    int merge_team;                      // warps that join a row's partial results
    float* scores;                       // [sequence, KV head][row][pitch], log2 frame, for the weights
    int64_t pitch;
    float* weights;                      // (B, KV_H, S)
    unsigned long long *begun, call;     // *begun == call: what ran before this call is complete, and so is what its earlier launches wait for
};

// Launches that begin beside the launch ahead of them, whose results they do not need.  That launch tells, behind its own wait, that what ran
// before is complete (one CTA of it, ahead of letting others begin); where nothing is told yet, as when another thread's launch came in between on the stream,
// the launch waits first, as all others do.  Either way it waits at its end: its end is the end of what lies before it.
__device__ __forceinline__ void tell_begun(const Params& P) {                 // (a release: what the wait made visible to this thread goes ahead of the word)
    asm volatile("st.release.gpu.global.u64 [%0], %1;" ::"l"(P.begun), "l"(P.call) : "memory");
}
__device__ __forceinline__ void wait_unless_begun(const Params& P) {
    unsigned long long told;
    asm volatile("ld.acquire.gpu.global.u64 %0, [%1];" : "=l"(told) : "l"(P.begun) : "memory");
    if (told != P.call) pdl_wait();
}
__device__ __forceinline__ void end_behind(const Params& P, bool last) {
    pdl_wait();
    if (last) *static_cast<volatile unsigned long long*>(P.begun) = 0;       // a graph's next replay begins anew
}

// One sequence of a call (pos: the row of the launch's first token): the keys its tokens tok0 .. tok1 - 1 see, as one run of `keys` places: `sink` first rows, then rows from lo on.
struct Seq {
    int pos, lo, sink, keys;
    __device__ __forceinline__ int row_of(int place) const { return place < sink ? place : lo + place - sink; }
};
__device__ __forceinline__ int live_pos(const Params& P, int b, bool tell) {
    const int pos = __ldcg(P.pos + (P.pos_count == 1 ? 0 : b));
    if (pos < 0) return -1;                                  // a sequence without tokens in this call
    if (pos > P.S - P.n_all) {
        if (tell) atomicOr(&g_span_status, SPAN_POS_RANGE);
        return -1;
    }
    return pos + P.tok0;
}
__device__ __forceinline__ Seq seq_at(const Params& P, int pos, int tok0, int tok1) {
    Seq s = {pos, 0, 0, 0};
    if (pos < 0) return s;
    if (P.window > 0) s.lo = max(0, pos + tok0 - P.window + 1);
    s.sink = min(P.sinks, s.lo);
    s.keys = s.sink + pos + tok1 - s.lo;
    return s;
}
__device__ __forceinline__ bool sees(const Params& P, int row_pos, int j) {
    return j <= row_pos && (P.window <= 0 || j > row_pos - P.window || j < P.sinks);
}

// The lowest n bits (none for n <= 0, all from 32 on).
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u); }

__device__ __forceinline__ uint32_t s32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Byte offset of 16-byte piece c of row r in a tile of D halves a row: eight rows' equal pieces fall into different banks.
template <int D>
__device__ __forceinline__ uint32_t piece_at(int r, int c) { return r * (D * 2) + ((c ^ (r & 7)) << 4); }

// Sixteen rows (a warp) or 64 rows and more (a CTA of `lanes` threads) of a tile, from rows that lie in one piece.  at: address of the first row plus this
// thread's piece; dst: the tile.  Everything but the row is a constant of the thread, and the rows' distances are offsets of the instruction.
template <int D, int ROWS, int LANES>
struct Copy {
    static constexpr int PIECES = D / 8, STRIDE = LANES / PIECES, N = ROWS / STRIDE;       // rows apart, copies of a thread
    __device__ __forceinline__ static int row(int thread) { return thread / PIECES; }
    __device__ __forceinline__ static int col(int thread) { return thread % PIECES * 8; }
    __device__ __forceinline__ static uint32_t place(int thread) { return piece_at<D>(row(thread), thread % PIECES); }
    __device__ __forceinline__ static void rows(uint32_t dst, const __half* at) {          // dst: the tile plus place()
#pragma unroll
        for (int i = 0; i < N; ++i)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((dst ^ ((i * STRIDE & 7) << 4)) + i * STRIDE * D * 2), "l"(at + i * STRIDE * D) : "memory");
    }
};

// Four consecutive outputs, each rounded once from fp32.
__device__ __forceinline__ void store4(void* out, int dtype, int64_t i, float a, float b, float c, float d) {
    uint2 w;
    if (dtype == ALLOYB_F16) {
        w = make_uint2(pack_h2(a, b), pack_h2(c, d));
    } else {
        const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
        w = make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i) = w;
}

__device__ __forceinline__ void store2(void* out, int dtype, int64_t i, float a, float b) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
    *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(out) + i) = dtype == ALLOYB_F16 ? pack_h2(a, b) : *reinterpret_cast<const uint32_t*>(&x);
}

// A query row on its way into shared memory as fp16, a warp's lanes D / 32 elements each.  Reading and placing are apart so that a warp
// asks for several rows before it waits for the first.
template <int D>
struct QRow {
    static constexpr int E = D / 32;
    uint32_t w[E / 2];
    __device__ __forceinline__ void read(const void* q, int64_t at, bool vec, bool live, int lane) {
#pragma unroll
        for (int e = 0; e < E / 2; ++e) w[e] = 0u;
        if (!live) return;                                   // rows past the last are zeros
        const uint16_t* src = static_cast<const uint16_t*>(q) + at + lane * E;
        if (vec) {
            if (E == 2) w[0] = __ldcg(reinterpret_cast<const uint32_t*>(src));
            if (E == 4) {
                const uint2 x = __ldcg(reinterpret_cast<const uint2*>(src));
                w[0] = x.x;
                w[1 % (E / 2)] = x.y;
            }
            if (E == 8) {
                const uint4 x = __ldcg(reinterpret_cast<const uint4*>(src));
                w[0] = x.x;
                w[1 % (E / 2)] = x.y;
                w[2 % (E / 2)] = x.z;
                w[3 % (E / 2)] = x.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < E / 2; ++e) w[e] = __ldcg(src + 2 * e) | static_cast<uint32_t>(__ldcg(src + 2 * e + 1)) << 16;
        }
    }
    // place(d): the shared address of element d.  bf16 rows are brought under 2^15 by a power of two, so that fp16 holds every element of at
    // least 2^-29 of the row's largest exactly; returns the factor that puts the row's scores back.
    template <typename Place>
    __device__ __forceinline__ float put(const Place& place, int dtype, int lane) {
        float back = 1.0f;
        if (dtype == ALLOYB_BF16) {
            float x[E], top = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                x[e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
                top = fmaxf(top, fabsf(x[e]));
            }
            top = warp_max(top);
            const int ex = static_cast<int>(__float_as_uint(top) >> 23);
            if (ex > 0 && ex < 255) {
                const int field = min(268 - ex, 253);        // 2^(field - 127): the largest element lands in [2^14, 2^15)
                const float f = __uint_as_float(static_cast<uint32_t>(field) << 23);
                back = __uint_as_float(static_cast<uint32_t>(254 - field) << 23);
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] *= f;
            }
#pragma unroll
            for (int e = 0; e < E / 2; ++e) w[e] = pack_h2(x[2 * e], x[2 * e + 1]);
        }
        const uint32_t to = place(lane * E);
        if (E == 2) asm volatile("st.shared.u32 [%0], %1;" ::"r"(to), "r"(w[0]) : "memory");
        if (E == 4) asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(to), "r"(w[0]), "r"(w[1 % (E / 2)]) : "memory");
        if (E == 8) asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(w[0]), "r"(w[1 % (E / 2)]), "r"(w[2 % (E / 2)]), "r"(w[3 % (E / 2)]) : "memory");
        return back;
    }
};

// A warp's sixteen rows against NK * 16 keys of a tile: running maximum m, sum l (this lane's columns only; times 64) and output o of rows
// g and g + 8, columns 8 i + 2 t of block i.
template <int D>
struct Rows {
    float m[2], l[2];
    float o[D / 8][4];
    __device__ __forceinline__ void clear() {
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    }
    // A lane's place in a 16 x 16 block of a tile (rows of D halves, piece_at order), as an A operand, a B operand (K) and a transposed B operand
    // (V).  Block c along the row is the same place with c << 5 exclusive-ored in: tiles begin on a multiple of their row's bytes.
    __device__ __forceinline__ static uint32_t a_lane(int lane) { return piece_at<D>((lane & 7) + ((lane >> 3) & 1) * 8, (lane >> 4) & 1); }
    __device__ __forceinline__ static uint32_t k_lane(int lane) { return piece_at<D>((lane & 7) + ((lane >> 4) & 1) * 8, (lane >> 3) & 1); }
    __device__ __forceinline__ static uint32_t v_lane(int lane) { return piece_at<D>((lane & 7) + ((lane >> 3) & 1) * 8, (lane >> 4) & 1); }
    __device__ __forceinline__ static void load_q(uint32_t (&q)[D / 16][4], uint32_t q_at) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) ldsm_x4(q_at ^ (kk << 5), q[kk]);
    }
    // S = Q K^T; k_at: the tile's address plus k_lane.  q: the fragments, or (null) read from q_at as they are used
    template <int NK>
    __device__ __forceinline__ static void scores(float (&s)[2 * NK][4], const uint32_t (*q)[4], uint32_t q_at, uint32_t k_at) {
#pragma unroll
        for (int n = 0; n < 2 * NK; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t a[4];
            if (q) {
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] = q[kk][e];
            } else {
                ldsm_x4(q_at ^ (kk << 5), a);
            }
#pragma unroll
            for (int n2 = 0; n2 < NK; ++n2) {
                uint32_t b[4];
                ldsm_x4((k_at ^ (kk << 5)) + n2 * 16 * D * 2, b);
                mma16816(s[2 * n2], a, b[0], b[1]);
                mma16816(s[2 * n2 + 1], a, b[2], b[3]);
            }
        }
    }
    // s: scores in the log2 frame, -inf where a row does not see the key (a NaN score makes the row NaN); v_at: the tile's address plus v_lane
    template <int NK>
    __device__ __forceinline__ void take(float (&s)[2 * NK][4], uint32_t v_at) {
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2 * NK; ++n) {
            mx[0] = fmaxf(mx[0], fmaxf(s[n][0], s[n][1]));
            mx[1] = fmaxf(mx[1], fmaxf(s[n][2], s[n][3]));
        }
        float sub[2], alpha[2];
        bool grow = false;
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            mx[rr] = fmaxf(mx[rr], __shfl_xor_sync(0xffffffffu, mx[rr], 1));
            mx[rr] = fmaxf(mx[rr], __shfl_xor_sync(0xffffffffu, mx[rr], 2));
            alpha[rr] = 1.0f;
            if (mx[rr] > m[rr] + RESCALE_LOG2) {             // (also the first score: m is -inf)
                alpha[rr] = ex2(m[rr] - mx[rr]);
                m[rr] = mx[rr];
                grow = true;
            }
            sub[rr] = m[rr] == -INFINITY ? 0.f : P_BIAS_LOG2 - m[rr];
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                o[i][0] *= alpha[0];
                o[i][1] *= alpha[0];
                o[i][2] *= alpha[1];
                o[i][3] *= alpha[1];
            }
            l[0] *= alpha[0];
            l[1] *= alpha[1];
        }
#pragma unroll
        for (int k2 = 0; k2 < NK; ++k2) {
            // P enters the product as two fp16 halves, which keep 22 bits of a weight (as in the framework's other attention: a call's accuracy does
            // not go by how many rows it has); the sum l is of the unrounded weights
            uint32_t p[4], low[4];
#pragma unroll
            for (int nn = 0; nn < 2; ++nn) {
                const float (&x)[4] = s[2 * k2 + nn];
                const float p0 = ex2(x[0] + sub[0]), p1 = ex2(x[1] + sub[0]), p2 = ex2(x[2] + sub[1]), p3 = ex2(x[3] + sub[1]);
                l[0] += p0 + p1;
                l[1] += p2 + p3;
                p[2 * nn] = pack_h2(p0, p1);
                p[2 * nn + 1] = pack_h2(p2, p3);
                const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&p[2 * nn])), b = __half22float2(*reinterpret_cast<const __half2*>(&p[2 * nn + 1]));
                low[2 * nn] = pack_h2(p0 - a.x, p1 - a.y);
                low[2 * nn + 1] = pack_h2(p2 - b.x, p3 - b.y);
            }
#pragma unroll
            for (int n2 = 0; n2 < D / 16; ++n2) {
                uint32_t b[4];
                ldsm_x4_t((v_at ^ (n2 << 5)) + k2 * 16 * D * 2, b);
                mma16816(o[2 * n2], p, b[0], b[1]);
                mma16816(o[2 * n2 + 1], p, b[2], b[3]);
                mma16816(o[2 * n2], low, b[0], b[1]);
                mma16816(o[2 * n2 + 1], low, b[2], b[3]);
            }
        }
    }
    __device__ __forceinline__ void sum_lanes() {
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 1);
            l[rr] += __shfl_xor_sync(0xffffffffu, l[rr], 2);
        }
    }
};

}  // namespace sp
}  // namespace alloyb
