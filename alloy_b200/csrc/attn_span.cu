// Attention of query tokens over spans of an fp16 cache: a window with sinks, a shared prefix with an own rest, and the form that
// keeps the attention weights.  out = sum_j softmax_j(scale q k_j) v_j over the keys j that a row sees; softmax in the exp2 frame with a
// running maximum and sum, K and V read once.
//
// Few rows (one token, or as many as give 16 rows of a KV head; span_stream_kernel).  Bound: HBM, 4 D bytes a key for 4 D G n operations.
// Every sequence's keys are cut into steps of 64, all sequences' steps laid end to end and dealt out evenly to as many CTAs as the GPU
// holds at once, whatever the lengths: a CTA may finish one sequence and begin the next, and its rings of tiles run on.  A warp takes 16 of a
// step's keys through a ring of its own (cp.async, three tiles of K and V, no barrier but its own), S and P V on mma.sync with the rows
// padded to 16.  A (sequence, KV head) that one CTA covers is stored by it; the others' partial results go to a workspace and
// span_merge_kernel joins them.  32 sequences of 4096 keys each at positions 2000 .. 16300, 32/8 heads, head_dim 128: 91 us = 5.7 TB/s.
// Where there is little to do, clusters that join through distributed shared memory do it in one launch (span_cluster_kernel).
//
// More rows (chunks, and all the batch's rows over a shared prefix; span_rows_kernel).  Bound: mma.sync.  A CTA owns 64 (token, head) rows,
// a warp 16 of them, and tiles of 64 keys (32 at head_dim 256) that its warps share; the keys are split where the tiles alone leave SMs
// empty.  4 x 16 scored tokens looking back over 5000 to 8100 keys: 53 us of the call's 67, 48 % of the tensor pipe.  While P was one fp16 half, tiles of
// 32 keys and three CTAs an SM were slower (the call 68 -> 81 us), a third stage gave nothing, and with a step's scores a step ahead of its softmax it
// took 70 -> 82.  Many rows with much to do go to attn_span_tc.cu.
//
// The weights (scored form): the scores are left in the workspace (4 bytes a row and key beside the 4 D that a key's K and V cost) and a
// launch of its own adds up exp2(score - the row's log-sum) over a KV head's rows, which needs no second read of K.  It joins the log-sums itself, so the
// outputs are joined beside it (the call above, with one half of P: 67 -> 60 us).
//
// New tokens' rows: keys from `pos` on are read from new_k / new_v, by every CTA that needs them, and written to the cache by one; nobody reads
// them there in the same launch.
#include <atomic>

#include "attn_span.cuh"

namespace alloyb {

// defined in attn_span_tc.cu
int launch_span_tc(const sp::Params& P, int D, bool prefix, dim3 grid, cudaStream_t st);
cudaError_t span_tc_status(int* status, int clear);

namespace sp {

// ---------------------------------------------------------------------------------------------------------------- few rows
template <int D>
struct StreamCfg {
    static constexpr int SLOTS = D == 64 ? 4 : 3;
    static constexpr int TILE = 16 * D * 2, SLOT = 2 * TILE;             // K, then V
    static constexpr int RING = WARPS * SLOTS * SLOT, OUT = WARPS * 16 * D * 4;
    static constexpr int Q = 16 * D * 2;
    static constexpr int SMEM = (RING > OUT ? RING : OUT) + Q;
};

// A CTA takes at least this many steps: fewer would give more partial results than they save time.
constexpr int MIN_STEPS = 2;

__device__ __forceinline__ int steps_per_cta(int total, int ctas) { return max((total + ctas - 1) / ctas, MIN_STEPS); }

// Requests places [place0, place0 + ROWS) of a span: K's rows to dst, V's `v_off` bytes behind; LANES threads, this one is `thread`.  Rows in one
// piece of the cache take the short way; the others (first rows next to the window, the sequence's end, new tokens) are told apart one by one,
// places past the last key are filled with zeros: what the cache holds there is nobody's business.
template <int D, int ROWS, int LANES>
__device__ __forceinline__ void request_span(const Params& P, const Seq& sq, int b, int kvh, int place0, uint32_t dst, uint32_t v_off, int thread) {
    using C = Copy<D, ROWS, LANES>;
    if (place0 >= sq.keys) return;                                       // (a warp's share of a last step: nobody looks at it)
    const int64_t head = (static_cast<int64_t>(b) * P.KV_H + kvh) * P.S * D;
    const int first = sq.row_of(place0);
    if (place0 + ROWS <= sq.keys && sq.row_of(place0 + ROWS - 1) == first + ROWS - 1 && (!P.nk || first + ROWS <= sq.pos)) {
        const int64_t at = head + static_cast<int64_t>(first + C::row(thread)) * D + C::col(thread);
        C::rows(dst + C::place(thread), P.k + at);
        C::rows(dst + v_off + C::place(thread), P.v + at);
        return;
    }
#pragma unroll 2
    for (int i = 0; i < C::N; ++i) {
        const int r = C::row(thread) + i * C::STRIDE, place = place0 + r;
        const bool live = place < sq.keys;
        const int j = live ? sq.row_of(place) : 0;
        int64_t from = head + static_cast<int64_t>(j) * D;
        const __half *k = P.k, *v = P.v;
        if (P.nk && live && j >= sq.pos) {
            from = b * P.n_bs + kvh * P.n_hs + (j - sq.pos) * P.n_ts;
            k = P.nk;
            v = P.nv;
        }
        const uint32_t to = dst + piece_at<D>(r, C::col(thread) / 8);
        copy16(to, k + from + C::col(thread), live);
        copy16(to + v_off, v + from + C::col(thread), live);
    }
}

// What the warps of a CTA leave for its epilogue.
struct StreamShared {
    float back[16], m[WARPS][16], l[WARPS][16];
};

// `steps` steps of one (sequence, KV head) from step0 on: maxima, sums and outputs of the four warps into shared memory (outputs at sm_o,
// [warp][16][D], where the rings were).  put(row, place, two scores) takes the scores.  A barrier is behind the last store.
template <int D, bool SCORED, typename Put>
__device__ __forceinline__ void span_segment(const Params& P, StreamShared& sh, uint8_t* smem, int b, int kvh, const Seq& sq, int step0, int steps, const Put& put) {
    using C = StreamCfg<D>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int rows = P.n * P.G;
    const uint32_t q_s = s32(smem), ring = q_s + C::Q + warp * (C::SLOTS * C::SLOT);
    float* sm_o = reinterpret_cast<float*>(smem + C::Q);

    auto request = [&](int i) {                                      // this warp's keys of the segment's i-th step
        if (i < steps) request_span<D, 16, 32>(P, sq, b, kvh, (step0 + i) * STEP + warp * 16, ring + i % C::SLOTS * C::SLOT, C::TILE, lane);
        copy_commit();
    };
#pragma unroll
    for (int i = 0; i < C::SLOTS - 1; ++i) request(i);
    // the rows of this (sequence, KV head); rows past the last are zero
    QRow<D> qr[16 / WARPS];
#pragma unroll
    for (int i = 0; i < 16 / WARPS; ++i) {
        const int r = warp + i * WARPS, tok = r / P.G, hg = r - tok * P.G;
        qr[i].read(P.q, b * P.q_bs + (kvh * P.G + hg) * P.q_hs + tok * P.q_ts, P.q_vec != 0, r < rows, lane);
    }
#pragma unroll
    for (int i = 0; i < 16 / WARPS; ++i) {
        const int r = warp + i * WARPS;
        const float f = qr[i].put([&](int d) { return q_s + piece_at<D>(r, d >> 3) + (d & 7) * 2; }, P.q_dtype, lane);
        if (lane == 0) sh.back[r] = f * P.scale_log2;
    }
    __syncthreads();
    const float scale[2] = {sh.back[g], sh.back[g + 8]};
    const int row_pos[2] = {sq.pos + g / P.G, sq.pos + (g + 8) / P.G};

    Rows<D> st;
    st.clear();
    for (int i = 0; i < steps; ++i) {
        request(i + C::SLOTS - 1);
        copy_wait<C::SLOTS - 1>();
        __syncwarp();
        const int place0 = (step0 + i) * STEP + warp * 16;
        const uint32_t k_tile = ring + i % C::SLOTS * C::SLOT;
        if (place0 < sq.keys) {
            float s[2][4];
            Rows<D>::template scores<1>(s, nullptr, q_s + Rows<D>::a_lane(lane), k_tile + Rows<D>::k_lane(lane));
            const bool whole = P.n == 1 && place0 + 16 <= sq.keys;   // one token sees every key of its spans
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int place = place0 + 8 * n + 2 * t + (e & 1);
                    const bool seen = whole || (place < sq.keys && sees(P, row_pos[e >> 1], sq.row_of(place)));
                    s[n][e] = seen ? s[n][e] * scale[e >> 1] : -INFINITY;
                }
            if (SCORED) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int rr = 0; rr < 2; ++rr)
                        if (g + 8 * rr < rows && place0 + 8 * n + 2 * t < sq.keys)
                            put(g + 8 * rr, place0 + 8 * n + 2 * t, make_float2(s[n][2 * rr], s[n][2 * rr + 1]));
            }
            st.template take<1>(s, k_tile + C::TILE + Rows<D>::v_lane(lane));
        }
        __syncwarp();                                                // the slot has been read: the next request may fill it
    }
    st.sum_lanes();
    copy_wait<0>();
    __syncthreads();                                                 // every warp is done with its ring
    if (t == 0) {
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
            sh.m[warp][g + 8 * rr] = st.m[rr];
            sh.l[warp][g + 8 * rr] = st.l[rr];
        }
    }
#pragma unroll
    for (int rr = 0; rr < 2; ++rr)
        if (g + 8 * rr < rows) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                *reinterpret_cast<float2*>(sm_o + (warp * 16 + g + 8 * rr) * D + 8 * i + 2 * t) = make_float2(st.o[i][2 * rr], st.o[i][2 * rr + 1]);
        }
    __syncthreads();
}
// The four warps' results of row r, dims d .. d + 3, joined: outputs relative to `top`, `l` the sum (times 2^P_BIAS_LOG2, both).
template <int D>
__device__ __forceinline__ float4 join_warps(const StreamShared& sh, const float* sm_o, int r, int d, float& top, float& l) {
    top = sh.m[0][r];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sh.m[w][r]);
    l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        const float f = sh.m[w][r] == -INFINITY && sh.l[w][r] == 0.f ? 0.f : ex2(sh.m[w][r] - top);
        const float4 x = *reinterpret_cast<const float4*>(sm_o + (w * 16 + r) * D + d);
        l = fmaf(f, sh.l[w][r], l);
        acc.x = fmaf(f, x.x, acc.x);
        acc.y = fmaf(f, x.y, acc.y);
        acc.z = fmaf(f, x.z, acc.z);
        acc.w = fmaf(f, x.w, acc.w);
    }
    return acc;
}
// The new rows of one (sequence, KV head) into the cache.
template <int D>
__device__ __forceinline__ void append_rows(const Params& P, int b, int kvh, int pos) {
    for (int e = threadIdx.x; e < P.n * (D / 8); e += WARPS * 32) {
        const int tok = e / (D / 8), c = (e - tok * (D / 8)) * 8;
        const int64_t src = b * P.n_bs + kvh * P.n_hs + tok * P.n_ts + c, dst = ((static_cast<int64_t>(b) * P.KV_H + kvh) * P.S + pos + tok) * D + c;
        *reinterpret_cast<uint4*>(P.k + dst) = ld_after_wait(P.nk + src);
        *reinterpret_cast<uint4*>(P.v + dst) = ld_after_wait(P.nv + src);
    }
}

// One place in a CTA's run of steps: a step of an item, i.e. of a (sequence, KV head).
struct Cursor {
    int b, kvh, step, steps;                                             // steps of the item
    Seq sq;
    __device__ __forceinline__ void enter(const Params& P) {             // sequence b, or the next that is not empty
        for (; b < P.B; ++b) {
            sq = seq_at(P, live_pos(P, b, false), 0, P.n);
            steps = (sq.keys + STEP - 1) / STEP;
            if (steps > 0) return;
        }
        b = P.B - 1;                                                     // (never, unless the positions change under the kernel)
        sq.keys = 0;
        steps = 1 << 30;
    }
    __device__ __forceinline__ void next_item(const Params& P) {
        step = 0;
        if (++kvh == P.KV_H) {
            kvh = 0;
            ++b;
            enter(P);
        }
    }
};

// Columns of the outputs that the warps join at a time, and where: rows of 64 floats, groups of eight permuted so that a warp's stores of
// eight rows spread over the banks.
constexpr int JOIN_COLS = 64, JOIN_BYTES = WARPS * 16 * JOIN_COLS * 4;
__device__ __forceinline__ int join_at(int w, int r, int c) { return (w * 16 + r) * JOIN_COLS + (c ^ ((r & 3) << 3)); }

template <int D>
struct RunCfg {
    static constexpr int SLOTS = 3, TILE = 16 * D * 2, SLOT = 2 * TILE;
    static constexpr int SMEM = JOIN_BYTES + WARPS * SLOTS * SLOT;       // the rows of q lie where the outputs are joined
};

// CTA `cta` of `ctas` over the steps of all items, an equal share each.  The rings run on from one item into the next.
template <int D, bool SCORED, bool PREFIX>
__device__ __forceinline__ void span_stream(const Params& P, int cta, int ctas) {
    using C = RunCfg<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ StreamShared sh;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int rows = P.n * P.G;
    const uint32_t q_s = s32(smem), ring = q_s + JOIN_BYTES + warp * (C::SLOTS * C::SLOT);
    float* sm_o = reinterpret_cast<float*>(smem);
    // steps before each sequence (every warp on its own): the total, then where this CTA's share begins
    int total = 0, begin = 0, end = 0, b0 = 0, before = 0;
    for (int pass = 0; pass < 2; ++pass) {
        int sum = 0;
        int next = lane < P.B ? live_pos(P, lane, cta == 0 && pass == 0 && warp == 0) : -1;
        for (int i0 = 0; i0 < P.B; i0 += 32) {
            const int b = i0 + lane, own = (seq_at(P, next, 0, P.n).keys + STEP - 1) / STEP * P.KV_H;
            next = b + 32 < P.B ? live_pos(P, b + 32, cta == 0 && pass == 0 && warp == 0) : -1;      // (asked for a round ahead)
            int upto = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            upto += sum;
            if (pass == 1) {
                if (cta == 0 && warp == 0 && b < P.B) P.cum[b + 1] = upto;
                const uint32_t here = __ballot_sync(0xffffffffu, upto - own <= begin && begin < upto);
                if (here) {
                    b0 = i0 + __ffs(here) - 1;
                    before = __shfl_sync(0xffffffffu, upto - own, __ffs(here) - 1);
                }
            }
            sum = __shfl_sync(0xffffffffu, upto, 31);
        }
        if (pass == 0) {
            total = sum;
            const int per = steps_per_cta(total, ctas);
            begin = min(total, cta * per);
            end = min(total, begin + per);
        }
    }
    if (cta == 0 && threadIdx.x == 0) P.cum[0] = 0;
    if (P.nk) {
        for (int i = cta; i < P.B * P.KV_H; i += ctas) {
            const int b = i / P.KV_H, pos = live_pos(P, b, false);
            if (pos >= 0) append_rows<D>(P, b, i - b * P.KV_H, pos);
        }
    }
    const int count = end - begin;
    if (count <= 0) return;
    Cursor rq, at;                                                       // the next step to request, the next to work on
    rq.b = b0;
    rq.enter(P);
    rq.kvh = (begin - before) / rq.steps;
    rq.step = begin - before - rq.kvh * rq.steps;
    at = rq;

    int requested = 0, slot_rq = 0, slot_at = 0;
    auto request = [&] {                                                 // this warp's sixteen keys of the next step
        if (requested < count) {
            request_span<D, 16, 32>(P, rq.sq, rq.b, rq.kvh, rq.step * STEP + warp * 16, ring + slot_rq * C::SLOT, C::TILE, lane);
            slot_rq = slot_rq + 1 == C::SLOTS ? 0 : slot_rq + 1;
            ++requested;
            if (++rq.step == rq.steps && requested < count) rq.next_item(P);
        }
        copy_commit();
    };
    QRow<D> qr[16 / WARPS];
    auto read_q = [&](const Cursor& c) {
#pragma unroll
        for (int i = 0; i < 16 / WARPS; ++i) {
            const int r = warp + i * WARPS, tok = r / P.G, hg = r - tok * P.G;
            qr[i].read(P.q, c.b * P.q_bs + (c.kvh * P.G + hg) * P.q_hs + tok * P.q_ts, P.q_vec != 0, r < rows, lane);
        }
    };
    auto put_q = [&] {
#pragma unroll
        for (int i = 0; i < 16 / WARPS; ++i) {
            const int r = warp + i * WARPS;
            const float f = qr[i].put([&](int d) { return q_s + piece_at<D>(r, d >> 3) + (d & 7) * 2; }, P.q_dtype, lane);
            if (lane == 0) sh.back[r] = f * P.scale_log2;
        }
    };
    // the query fragments stay in registers for an item (head_dim 256: the outputs leave no room, they are read anew for every step)
    constexpr bool Q_REGS = D <= 128;
    uint32_t qf[Q_REGS ? D / 16 : 1][4];
    float scale[2];
    auto take_q = [&] {
        put_q();
        __syncthreads();
        scale[0] = sh.back[g];
        scale[1] = sh.back[g + 8];
        if constexpr (Q_REGS) Rows<D>::load_q(qf, q_s + Rows<D>::a_lane(lane));
    };
    read_q(at);
#pragma unroll 1
    for (int i = 0; i < C::SLOTS - 1; ++i) request();
    take_q();

    Rows<D> st;
    st.clear();
    int first = 0, first_step = at.step;                                 // of the segment: the share's step, the item's step
    for (int i = 0; i < count; ++i) {
        request();
        copy_wait<C::SLOTS - 1>();
        __syncwarp();
        const int place0 = at.step * STEP + warp * 16;
        const uint32_t k_tile = ring + slot_at * C::SLOT;
        slot_at = slot_at + 1 == C::SLOTS ? 0 : slot_at + 1;
        if (place0 < at.sq.keys) {
            float s[2][4];
            Rows<D>::template scores<1>(s, Q_REGS ? qf : nullptr, q_s + Rows<D>::a_lane(lane), k_tile + Rows<D>::k_lane(lane));
            const bool whole = P.n == 1 && place0 + 16 <= at.sq.keys;    // one token sees every key of its spans
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int place = place0 + 8 * n + 2 * t + (e & 1);
                    const bool seen = whole || (place < at.sq.keys && sees(P, at.sq.pos + (g + 8 * (e >> 1)) / P.G, at.sq.row_of(place)));
                    s[n][e] = seen ? s[n][e] * scale[e >> 1] : -INFINITY;
                }
            if (SCORED) {
                float* to = P.scores + static_cast<int64_t>(at.b * P.KV_H + at.kvh) * rows * P.pitch + place0 + 2 * t;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int rr = 0; rr < 2; ++rr)
                        if (g + 8 * rr < rows && place0 + 8 * n + 2 * t < at.sq.keys)
                            *reinterpret_cast<float2*>(to + (g + 8 * rr) * P.pitch + 8 * n) = make_float2(s[n][2 * rr], s[n][2 * rr + 1]);
            }
            st.template take<1>(s, k_tile + C::TILE + Rows<D>::v_lane(lane));
        }
        __syncwarp();                                                    // the slot has been read: the next request may fill it
        if (++at.step < at.steps && i + 1 < count) continue;

        // ---- the segment's end: the warps' results joined and stored, the next item's rows of q
        Cursor next = at;
        if (i + 1 < count) {
            next.next_item(P);
            read_q(next);
        }
        st.sum_lanes();
        if (t == 0) {
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
                sh.m[warp][g + 8 * rr] = st.m[rr];
                sh.l[warp][g + 8 * rr] = st.l[rr];
            }
        }
        __syncthreads();                                                 // every warp is done with q
        const int item = at.b * P.KV_H + at.kvh;
        const bool all = first_step == 0 && at.step == at.steps;
        const int64_t slot = all ? 2 * ctas + item : 2 * cta + (first > 0);
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += JOIN_COLS) {
            if (c0 > 0) __syncthreads();
#pragma unroll
            for (int rr = 0; rr < 2; ++rr)
                if (g + 8 * rr < rows) {
#pragma unroll
                    for (int x = 0; x < JOIN_COLS / 8; ++x)
                        *reinterpret_cast<float2*>(sm_o + join_at(warp, g + 8 * rr, 8 * x + 2 * t)) =
                            make_float2(st.o[c0 / 8 + x][2 * rr], st.o[c0 / 8 + x][2 * rr + 1]);
                }
            __syncthreads();
            for (int x = threadIdx.x; x < rows * (JOIN_COLS / 4); x += WARPS * 32) {
                const int r = x / (JOIN_COLS / 4), d = x % (JOIN_COLS / 4) * 4;
                float top = sh.m[0][r], l = 0.f;
#pragma unroll
                for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sh.m[w][r]);
                float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    const float f = sh.m[w][r] == -INFINITY && sh.l[w][r] == 0.f ? 0.f : ex2(sh.m[w][r] - top);
                    const float4 o = *reinterpret_cast<const float4*>(sm_o + join_at(w, r, d));
                    l = fmaf(f, sh.l[w][r], l);
                    acc = make_float4(fmaf(f, o.x, acc.x), fmaf(f, o.y, acc.y), fmaf(f, o.z, acc.z), fmaf(f, o.w, acc.w));
                }
                const float inv = l == 0.f ? 0.f : 1.0f / l;
                acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
                if (c0 + d == 0) P.part_lse[slot * 16 + r] = l == 0.f ? -INFINITY : top + log2f(l) - P_BIAS_LOG2;
                if (all && !PREFIX) {
                    const int tok = r / P.G, hg = r - tok * P.G;
                    store4(P.out, P.q_dtype, ((static_cast<int64_t>(at.b) * P.n_all + tok) * P.H + at.kvh * P.G + hg) * D + c0 + d, acc.x, acc.y, acc.z, acc.w);
                } else {
                    *reinterpret_cast<float4*>(P.part_o + (slot * 16 + r) * D + c0 + d) = acc;
                }
            }
        }
        if (i + 1 == count) break;
        __syncthreads();                                                 // the join is over: q may lie there again
        take_q();
        at = next;
        st.clear();
        first = i + 1;
        first_step = 0;
    }
    copy_wait<0>();
}
template <int D, bool SCORED>
__global__ void __launch_bounds__(WARPS * 32, D == 64 ? 3 : (D == 128 ? 2 : 1)) span_stream_kernel(const Params P) {
    pdl_launch_dependents();
    pdl_wait();
    span_stream<D, SCORED, false>(P, blockIdx.x, gridDim.x);
}

// Few (sequence, KV head)s of few keys: a cluster of CTAs each, joined through distributed shared memory, all in one launch.  The scored
// form keeps its scores in shared memory ([row][the CTA's keys]) and needs nothing of the workspace.
__device__ __forceinline__ uint32_t peer_addr(const void* p, int rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(s32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ float peer_f32(const float* p, int rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ float4 peer_f32x4(const float* p, int rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer_addr(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Grid (CTAs of a cluster, B * KV_H); P.splits CTAs a cluster, P.tiles steps at most a CTA.
template <int D, bool SCORED>
__global__ void __launch_bounds__(WARPS * 32) span_cluster_kernel(const Params P) {
    using C = StreamCfg<D>;
    pdl_launch_dependents();
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ StreamShared sh;
    __shared__ float cta_m[16], cta_l[16], lse[16];
    const int item = blockIdx.y, b = item / P.KV_H, kvh = item - b * P.KV_H, rank = blockIdx.x, ranks = P.splits;
    const int rows = P.n * P.G;
    float* sm_o = reinterpret_cast<float*>(smem + C::Q);
    float* sm_s = reinterpret_cast<float*>(smem + C::SMEM);              // scored: [row][tiles * STEP]
    pdl_wait();
    const int pos = live_pos(P, b, rank == 0 && kvh == 0 && threadIdx.x == 0);
    if (P.nk && rank == ranks - 1 && pos >= 0) append_rows<D>(P, b, kvh, pos);
    const Seq sq = seq_at(P, pos, 0, P.n);
    const int total = (sq.keys + STEP - 1) / STEP, per = (total + ranks - 1) / ranks;
    const int step0 = min(total, rank * per), steps = min(total, step0 + per) - step0;
    span_segment<D, SCORED>(P, sh, smem, b, kvh, sq, step0, steps, [&](int r, int place, float2 s) {
        *reinterpret_cast<float2*>(sm_s + r * (P.tiles * STEP) + place - step0 * STEP) = s;
    });
    for (int i = threadIdx.x; i < rows * (D / 4); i += WARPS * 32) {
        const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
        float top, l;
        const float4 acc = join_warps<D>(sh, sm_o, r, d, top, l);
        *reinterpret_cast<float4*>(sm_o + r * D + d) = acc;              // (warp 0's place: nobody else reads it)
        if (d == 0) {
            cta_m[r] = top;
            cta_l[r] = l;
        }
    }
    cluster_barrier();
    for (int i = rank + threadIdx.x * ranks; i < rows * (D / 4); i += WARPS * 32 * ranks) {
        const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
        float top = -INFINITY, l = 0.f;
        for (int k = 0; k < ranks; ++k) top = fmaxf(top, peer_f32(cta_m + r, k));
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < ranks; ++k) {
            const float m = peer_f32(cta_m + r, k), lk = peer_f32(cta_l + r, k), f = m == -INFINITY && lk == 0.f ? 0.f : ex2(m - top);
            const float4 x = peer_f32x4(sm_o + r * D + d, k);
            l = fmaf(f, lk, l);
            acc = make_float4(fmaf(f, x.x, acc.x), fmaf(f, x.y, acc.y), fmaf(f, x.z, acc.z), fmaf(f, x.w, acc.w));
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        const int tok = r / P.G, hg = r - tok * P.G;
        store4(P.out, P.q_dtype, ((static_cast<int64_t>(b) * P.n_all + tok) * P.H + kvh * P.G + hg) * D + d, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
    if (SCORED) {
        if (threadIdx.x < rows) {
            float top = -INFINITY, l = 0.f;
            for (int k = 0; k < ranks; ++k) top = fmaxf(top, peer_f32(cta_m + threadIdx.x, k));
            for (int k = 0; k < ranks; ++k) {
                const float m = peer_f32(cta_m + threadIdx.x, k), lk = peer_f32(cta_l + threadIdx.x, k);
                l += m == -INFINITY && lk == 0.f ? 0.f : lk * ex2(m - top);
            }
            lse[threadIdx.x] = l == 0.f ? INFINITY : top + log2f(l) - P_BIAS_LOG2;      // (a row whose scores are all -inf adds nothing)
        }
        __syncthreads();
        float* w = P.weights + static_cast<int64_t>(item) * P.S;
        for (int i = threadIdx.x; i < steps * STEP && step0 * STEP + i < sq.keys; i += WARPS * 32) {
            const int j = step0 * STEP + i;
            float sum = 0.f;
            for (int r = 0; r < rows; ++r) sum += ex2(sm_s[r * (P.tiles * STEP) + i] - lse[r]);
            if (j < pos) sum += __ldcg(w + j);
            w[j] = sum;
        }
    }
    cluster_barrier();                                                   // nobody's shared memory goes away while a peer still reads it
}

// ---------------------------------------------------------------------------------------------------------------- more rows
template <int D>
struct RowsCfg {
    static constexpr int KT = D == 256 ? 32 : 64, STAGES = 2;
    static constexpr int Q = 64 * D * 2, TILE = KT * D * 2;
    static constexpr int SMEM = Q + STAGES * 2 * TILE;
};

// One CTA of a tile: `split` of `splits` CTAs that share its keys.  PREFIX: rows of the whole batch over the shared prefix, partial results only.
template <int D, bool SCORED, bool PREFIX>
__device__ __forceinline__ void span_rows(const Params& P, int tile, int tiles, int split, int splits, int kvh, int b) {
    using C = RowsCfg<D>;
    constexpr int KT = C::KT;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ float back[64];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int rows = P.n * P.G, all_rows = PREFIX ? rows * P.B : rows, row0 = tile * 64;
    const uint32_t q_s = s32(smem), tiles_s = q_s + C::Q;
    const int tok0 = row0 / P.G, tok1 = min(P.n, (row0 + 63) / P.G + 1);                // of a chunk: the tokens of these rows
    Seq sq = {0, 0, 0, P.P};
    if (!PREFIX) sq = seq_at(P, live_pos(P, b, tile == 0 && kvh == 0 && split == 0 && threadIdx.x == 0), tok0, tok1);
    const int steps = (sq.keys + KT - 1) / KT, per = (steps + splits - 1) / splits;
    const int step0 = min(steps, split * per), step1 = min(steps, step0 + per);
    const int64_t head = (static_cast<int64_t>(b) * P.KV_H + kvh) * P.S * D;

    auto request = [&](int step) {
        if (step < step1) {
            const uint32_t dst = tiles_s + (step - step0) % C::STAGES * (2 * C::TILE);
            if (!PREFIX) {
                request_span<D, KT, WARPS * 32>(P, sq, b, kvh, step * KT, dst, C::TILE, threadIdx.x);
            } else {
                using Rq = Copy<D, KT, WARPS * 32>;
                const int64_t at = kvh * P.p_hs + static_cast<int64_t>(step * KT + Rq::row(threadIdx.x)) * D + Rq::col(threadIdx.x);
                if (step * KT + KT <= P.P) {
                    Rq::rows(dst + Rq::place(threadIdx.x), P.pk + at);
                    Rq::rows(dst + C::TILE + Rq::place(threadIdx.x), P.pv + at);
                } else {
#pragma unroll 2
                    for (int i = 0; i < Rq::N; ++i) {
                        const int r = Rq::row(threadIdx.x) + i * Rq::STRIDE;
                        const bool live = step * KT + r < P.P;
                        const int64_t from = live ? at + static_cast<int64_t>(i) * Rq::STRIDE * D : 0;
                        const uint32_t to = dst + piece_at<D>(r, Rq::col(threadIdx.x) / 8);
                        copy16(to, P.pk + from, live);
                        copy16(to + C::TILE, P.pv + from, live);
                    }
                }
            }
        }
        copy_commit();
    };
    request(step0);
    if (!PREFIX && P.nk && split == 0 && sq.pos >= 0) {
        // the tokens whose first row is in this tile: their new rows into the cache
        const int ta = (row0 + P.G - 1) / P.G, tb = min(P.n, (row0 + 63) / P.G + 1);
        for (int e = threadIdx.x; e < (tb - ta) * (D / 8); e += WARPS * 32) {
            const int tok = ta + e / (D / 8), c = (e % (D / 8)) * 8;
            const int64_t src = b * P.n_bs + kvh * P.n_hs + tok * P.n_ts + c, dst = head + static_cast<int64_t>(sq.pos + tok) * D + c;
            *reinterpret_cast<uint4*>(P.k + dst) = ld_after_wait(P.nk + src);
            *reinterpret_cast<uint4*>(P.v + dst) = ld_after_wait(P.nv + src);
        }
    }
#pragma unroll 1
    for (int i0 = 0; i0 < 64 / WARPS; i0 += 8) {
        QRow<D> qr[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int R = row0 + warp + (i0 + i) * WARPS, rb = PREFIX ? R / rows : b, rest = PREFIX ? R - rb * rows : R, tok = rest / P.G, hg = rest - tok * P.G;
            qr[i].read(P.q, rb * P.q_bs + (kvh * P.G + hg) * P.q_hs + tok * P.q_ts, P.q_vec != 0, R < all_rows, lane);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = warp + (i0 + i) * WARPS;
            const float f = qr[i].put([&](int d) { return q_s + piece_at<D>(r, d >> 3) + (d & 7) * 2; }, P.q_dtype, lane);
            if (lane == 0) back[r] = f * P.scale_log2;
        }
    }
    __syncthreads();
    const int r_own[2] = {row0 + warp * 16 + g, row0 + warp * 16 + g + 8};
    const float scale[2] = {back[warp * 16 + g], back[warp * 16 + g + 8]};
    const int row_pos[2] = {sq.pos + r_own[0] / P.G, sq.pos + r_own[1] / P.G};
    const int first = sq.pos + (row0 + warp * 16) / P.G, last = sq.pos + (row0 + warp * 16 + 15) / P.G;   // the warp's earliest and latest row
    const int item = b * P.KV_H + kvh;

    Rows<D> st;
    st.clear();
    for (int step = step0; step < step1; ++step) {
        request(step + 1);
        copy_wait<1>();
        __syncthreads();
        const uint32_t k_tile = tiles_s + (step - step0) % C::STAGES * (2 * C::TILE);
        float s[KT / 8][4];
        Rows<D>::template scores<KT / 16>(s, nullptr, q_s + warp * 16 * D * 2 + Rows<D>::a_lane(lane), k_tile + Rows<D>::k_lane(lane));
        const int place0 = step * KT;
        bool whole = place0 + KT <= sq.keys;
        if (!PREFIX && whole) {
            // every row of the warp sees every key: none lies behind the earliest row, and none before the latest row's window
            const int j0 = sq.row_of(place0), j1 = sq.row_of(place0 + KT - 1);
            whole = j1 <= first && (P.window <= 0 || (place0 >= sq.sink && j0 > last - P.window) || (place0 + KT <= sq.sink));
        }
        if (whole) {
#pragma unroll
            for (int n = 0; n < KT / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] *= scale[e >> 1];
        } else {
#pragma unroll
            for (int n = 0; n < KT / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int place = place0 + 8 * n + 2 * t + (e & 1);
                    const bool seen = place < sq.keys && (PREFIX || sees(P, row_pos[e >> 1], sq.row_of(place)));
                    s[n][e] = seen ? s[n][e] * scale[e >> 1] : -INFINITY;
                }
        }
        if (SCORED) {
#pragma unroll
            for (int n = 0; n < KT / 8; ++n)
#pragma unroll
                for (int rr = 0; rr < 2; ++rr)
                    if (r_own[rr] < rows && place0 + 8 * n + 2 * t < sq.keys)
                        *reinterpret_cast<float2*>(P.scores + (static_cast<int64_t>(item) * rows + r_own[rr]) * P.pitch + place0 + 8 * n + 2 * t) =
                            make_float2(s[n][2 * rr], s[n][2 * rr + 1]);
        }
        st.template take<KT / 16>(s, k_tile + C::TILE + Rows<D>::v_lane(lane));
        __syncthreads();                                                 // the tile has been read: its stage may be refilled
    }
    copy_wait<0>();
    st.sum_lanes();
    const bool direct = !PREFIX && splits == 1 && P.pre_o == nullptr;
    const int64_t slot = ((static_cast<int64_t>(PREFIX ? 0 : b) * P.KV_H + kvh) * tiles + tile) * splits + split;
    float* po = PREFIX ? P.pre_o : P.part_o;
    float* pl = PREFIX ? P.pre_lse : P.part_lse;
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) {
        if (r_own[rr] >= all_rows) continue;
        const int r = warp * 16 + g + 8 * rr;
        const float inv = st.l[rr] == 0.f ? 0.f : 1.0f / st.l[rr];
        if (t == 0 && (!direct || SCORED)) pl[slot * 64 + r] = st.l[rr] == 0.f ? -INFINITY : st.m[rr] + log2f(st.l[rr]) - P_BIAS_LOG2;
        if (direct) {
            const int tok = r_own[rr] / P.G, hg = r_own[rr] - tok * P.G;
            const int64_t at = ((static_cast<int64_t>(b) * P.n_all + tok) * P.H + kvh * P.G + hg) * D;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                const float x = st.o[i][2 * rr] * inv, y = st.o[i][2 * rr + 1] * inv;
                if (P.q_dtype == ALLOYB_F16) *reinterpret_cast<__half2*>(static_cast<__half*>(P.out) + at + 8 * i + 2 * t) = __floats2half2_rn(x, y);
                else *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(P.out) + at + 8 * i + 2 * t) = __floats2bfloat162_rn(x, y);
            }
        } else {
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                *reinterpret_cast<float2*>(po + (slot * 64 + r) * D + 8 * i + 2 * t) = make_float2(st.o[i][2 * rr] * inv, st.o[i][2 * rr + 1] * inv);
        }
    }
}

// Grid (tiles * splits, KV_H, B); the rows with the most keys go first.
template <int D, bool SCORED>
__global__ void __launch_bounds__(WARPS * 32) span_rows_kernel(const Params P) {
    pdl_launch_dependents();
    pdl_wait();
    span_rows<D, SCORED, false>(P, P.tiles - 1 - blockIdx.x / P.splits, P.tiles, blockIdx.x % P.splits, P.splits, blockIdx.y, blockIdx.z);
}
// A shared prefix and the sequences' own keys in one launch: the first CTAs have the prefix, the last P.ctas the own keys (P.ctas 0: none,
// they are many rows and have a launch of their own).
template <int D>
__global__ void __launch_bounds__(WARPS * 32, D == 64 ? 3 : (D == 128 ? 2 : 1)) span_prefix_kernel(const Params P) {
    pdl_launch_dependents();
    pdl_wait();
    const int tiles = (P.B * P.n * P.G + 63) / 64, i = blockIdx.x, pre = static_cast<int>(gridDim.x) - P.ctas;
    if (i < pre) span_rows<D, false, true>(P, i / P.pre_splits % tiles, tiles, i % P.pre_splits, P.pre_splits, i / (P.pre_splits * tiles), 0);
    else span_stream<D, false, true>(P, i - pre, P.ctas);
}
// The own keys behind a prefix that the 5th-generation tensor cores have.  Nothing here reads what that kernel writes, so
// these CTAs take the SMs as those leave them (64 sequences of 64/8 heads over 32768 shared keys and up to 1000 of their own: 146 -> 134 us).
template <int D>
__global__ void __launch_bounds__(WARPS * 32, D == 64 ? 3 : (D == 128 ? 2 : 1)) span_stream_prefix_kernel(const Params P) {
    pdl_launch_dependents();
    wait_unless_begun(P);
    span_stream<D, false, true>(P, blockIdx.x, gridDim.x);
    end_behind(P, blockIdx.x == 0 && threadIdx.x == 0);
}

// ---------------------------------------------------------------------------------------------------------------- joining
constexpr int MERGE_WARPS = 8;
// Where the partial results of row R of a (sequence, KV head) lie.
struct Parts {
    int own, pre;                                                        // how many of the row's own keys, of the prefix
    int64_t own_at, own_step, own_first, pre_at;                         // indices (slot * rows of a slot + row) of part 0 / their distance
    bool stored;                                                         // the output is there already
    __device__ __forceinline__ int64_t own_index(int i) const { return i == 0 ? own_first : own_at + i * own_step; }
};
// (steps: of the sequences before this one, of them and it, of all)
template <bool STREAM>
__device__ __forceinline__ Parts parts_of(const Params& P, int b, int kvh, int R, const int (&steps)[3]) {
    Parts p;
    const bool prefix = P.pre_o != nullptr;
    const int item = b * P.KV_H + kvh;
    if (STREAM) {
        const int seq_steps = (steps[1] - steps[0]) / P.KV_H, per = steps_per_cta(steps[2], P.ctas), first = steps[0] + kvh * seq_steps;
        p.stored = false;
        if (seq_steps == 0) {
            p.own = 0;
        } else {
            const int a = first / per, z = (first + seq_steps - 1) / per;
            p.own = z - a + 1;
            p.own_first = (p.own == 1 ? 2 * static_cast<int64_t>(P.ctas) + item : 2 * static_cast<int64_t>(a) + (first > a * per)) * 16 + R;
            p.own_at = 2 * static_cast<int64_t>(a) * 16 + R;
            p.own_step = 2 * 16;
            p.stored = p.own == 1 && !prefix;
        }
    } else {
        p.own = P.splits;
        p.own_first = p.own_at = (static_cast<int64_t>(item) * P.tiles + R / P.tile_rows) * P.splits * P.tile_rows + R % P.tile_rows;
        p.own_step = P.tile_rows;
        p.stored = P.splits == 1 && !prefix;
    }
    p.pre = 0;
    if (prefix) {
        const int all = b * P.n * P.G + R, tr = P.pre_tile_rows, tiles = (P.B * P.n * P.G + tr - 1) / tr;
        p.pre = P.pre_splits;
        p.pre_at = (static_cast<int64_t>(kvh) * tiles + all / tr) * P.pre_splits * tr + all % tr;
    }
    return p;
}

// Steps before a sequence, of it and those before, of all.
__device__ __forceinline__ void steps_of(const Params& P, int b, int (&steps)[3]) {
    steps[0] = __ldcg(P.cum + b);
    steps[1] = __ldcg(P.cum + b + 1);
    steps[2] = __ldcg(P.cum + P.B);
}
// P.merge_team warps a row, 1 or all.
template <int D, bool STREAM>
__device__ __forceinline__ void join_rows(const Params& P) {
    __shared__ float4 sm[MERGE_WARPS * D / 4];                           // a warp's sums each
    __shared__ float sm_m[MERGE_WARPS], sm_l[MERGE_WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, item = blockIdx.y, rows = P.n * P.G;
    const int b = item / P.KV_H, kvh = item - b * P.KV_H;
    const int team = P.merge_team;
    int steps[3] = {0, 0, 0};
    if (STREAM) steps_of(P, b, steps);                                   // asked for along with the position, not behind it
    const int pos = live_pos(P, b, false);
    const int R = (blockIdx.x * MERGE_WARPS + warp) / team, w0 = warp % team;
    if (R >= rows) return;                                               // (a whole CTA's row, or a warp's: nobody waits for it)
    const Parts p = parts_of<STREAM>(P, b, kvh, R, steps);
    if (p.stored) return;
    // one pass: the parts' log-sums and outputs are asked for several at once, the running maximum and sum follow
    constexpr int E = D / 32 < 4 ? D / 32 : 4, PER = D / 32 / E;     // elements of a lane's access, accesses
    float m = -INFINITY, l = 0.f, acc[D / 32];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = 0.f;
    constexpr int AT_ONCE = D == 256 ? 4 : 8;
    if (pos >= 0) {
        for (int i0 = w0; i0 < p.own + p.pre; i0 += AT_ONCE * team) {
            float x[AT_ONCE], v[AT_ONCE][D / 32];
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const int i = i0 + k * team;
                const bool own = i < p.own, there = i < p.own + p.pre;
                const int64_t at = own ? p.own_index(i) : p.pre_at + static_cast<int64_t>(i - p.own) * P.pre_tile_rows;
                x[k] = there ? __ldcg((own ? P.part_lse : P.pre_lse) + at) : -INFINITY;
#pragma unroll
                for (int c = 0; c < PER; ++c) {
                    const float* src = (own ? P.part_o : P.pre_o) + at * D + (c * 32 + lane) * E;
                    if (E == 4) *reinterpret_cast<float4*>(v[k] + c * E) = there ? __ldcg(reinterpret_cast<const float4*>(src)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    else *reinterpret_cast<float2*>(v[k] + c * E) = there ? __ldcg(reinterpret_cast<const float2*>(src)) : make_float2(0.f, 0.f);
                }
            }
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const bool live = x[k] != -INFINITY;                     // (an empty part's outputs were never written)
                const float top = fmaxf(m, x[k]), f0 = m == -INFINITY ? 0.f : ex2(m - top), f1 = live ? ex2(x[k] - top) : 0.f;
                l = fmaf(l, f0, f1);
#pragma unroll
                for (int e = 0; e < D / 32; ++e) acc[e] = acc[e] * f0 + (live ? f1 * v[k][e] : 0.f);
                m = top;
            }
        }
    }
    const int tok = R / P.G, hg = R - tok * P.G;
    const int64_t out = ((static_cast<int64_t>(b) * P.n_all + tok) * P.H + kvh * P.G + hg) * D;
    if (team == 1) {
        const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
        for (int c = 0; c < PER; ++c) {
            const int64_t at = out + (c * 32 + lane) * E;
            if (E == 4) store4(P.out, P.q_dtype, at, acc[c * E] * inv, acc[c * E + 1] * inv, acc[c * E + 2 % E] * inv, acc[c * E + 3 % E] * inv);
            else store2(P.out, P.q_dtype, at, acc[c * E] * inv, acc[c * E + 1] * inv);
        }
        return;
    }
    float* sm_o = reinterpret_cast<float*>(sm);
    if (lane == 0) {
        sm_m[warp] = m;
        sm_l[warp] = l;
    }
#pragma unroll
    for (int c = 0; c < PER; ++c)
#pragma unroll
        for (int e = 0; e < E; ++e) sm_o[warp * D + (c * 32 + lane) * E + e] = acc[c * E + e];
    __syncthreads();
    if (threadIdx.x < D / 4) {
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < MERGE_WARPS; ++w) top = fmaxf(top, sm_m[w]);
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < MERGE_WARPS; ++w) {
            const float4 v = sm[w * (D / 4) + threadIdx.x];
            const float f = sm_m[w] == -INFINITY && sm_l[w] == 0.f ? 0.f : ex2(sm_m[w] - top);
            sum = fmaf(f, sm_l[w], sum);
            x = make_float4(fmaf(f, v.x, x.x), fmaf(f, v.y, x.y), fmaf(f, v.z, x.z), fmaf(f, v.w, x.w));
        }
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        store4(P.out, P.q_dtype, out + threadIdx.x * 4, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
    }
}

// Grid (CTAs for the rows, sequences * KV heads).  BESIDE: behind the weights' kernel, which reads the same partial results.
template <int D, bool STREAM, bool BESIDE>
__global__ void __launch_bounds__(MERGE_WARPS * 32) span_merge_kernel(const Params P) {
    pdl_launch_dependents();
    if (BESIDE) wait_unless_begun(P);
    else pdl_wait();
    join_rows<D, STREAM>(P);
    if (BESIDE) end_behind(P, blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0);
}

// The weights of the scored form: a CTA joins the rows' log-sums from their parts, and a thread adds up four keys' probabilities, of up to 16 rows
// (STREAM) all, of more a quarter, in a fixed order.  Grid (key chunks, sequences * KV heads).
template <bool STREAM>
struct Weights {
    static constexpr int THREADS = 256, GROUPS = STREAM ? 1 : 4, KEYS = THREADS * 4 / GROUPS;
};
template <bool STREAM>
__global__ void __launch_bounds__(256) span_weights_kernel(const Params P) {
    using W = Weights<STREAM>;
    __shared__ float4 sm[STREAM ? 1 : W::THREADS];
    __shared__ float lse[STREAM ? 16 : W::THREADS];
    const int item = blockIdx.y, b = item / P.KV_H, kvh = item - b * P.KV_H, rows = P.n * P.G, first_key = blockIdx.x * W::KEYS;
    const int group = threadIdx.x / (W::KEYS / 4), j0 = first_key + threadIdx.x % (W::KEYS / 4) * 4;
    float* weights = P.weights + static_cast<int64_t>(item) * P.S;
    const float* scores = P.scores + static_cast<int64_t>(item) * rows * P.pitch + j0;
    pdl_wait();
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        if (threadIdx.x == 0) tell_begun(P);
        __syncthreads();
    }
    pdl_launch_dependents();
    int steps[3] = {0, 0, 0};
    if (STREAM) steps_of(P, b, steps);
    const int pos = live_pos(P, b, false), len = pos + P.n;
    if (pos < 0 || first_key >= len) return;
    // the rows from r0 on, as many as fit
    auto join_lse = [&](int r0) {
        const int R = r0 + threadIdx.x;
        if (static_cast<int>(threadIdx.x) < (STREAM ? 16 : W::THREADS) && R < rows) {
            const Parts p = parts_of<STREAM>(P, b, kvh, R, steps);
            float m = -INFINITY, l = 0.f;
#pragma unroll 4
            for (int i = 0; i < p.own; ++i) {
                const float x = __ldcg(P.part_lse + p.own_index(i)), top = fmaxf(m, x);
                if (x == -INFINITY) continue;                            // (an empty part)
                l = l * (m == -INFINITY ? 0.f : ex2(m - top)) + ex2(x - top);    // (a NaN stays one)
                m = top;
            }
            lse[threadIdx.x] = l == 0.f ? INFINITY : m + log2f(l);       // (a row whose scores are all -inf adds nothing)
        }
        __syncthreads();
    };
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    for (int r0 = 0; r0 < rows; r0 += W::THREADS) {
        if (r0 > 0) __syncthreads();
        join_lse(r0);
        const int r1 = min(rows, r0 + W::THREADS);
        if (j0 + 3 <= pos) {                                             // every row sees the four keys
#pragma unroll 8
            for (int r = r0 + group; r < r1; r += W::GROUPS) {
                const float4 s = __ldcg(reinterpret_cast<const float4*>(scores + r * P.pitch));
                const float x = lse[r - r0];
                sum[0] += ex2(s.x - x);
                sum[1] += ex2(s.y - x);
                sum[2] += ex2(s.z - x);
                sum[3] += ex2(s.w - x);
            }
        } else if (j0 < len) {                                           // (a key behind the row's own position may have no score)
            for (int r = r0 + group; r < r1; r += W::GROUPS) {
                const float x = lse[r - r0];
                const int room = min(3, pos + r / P.G - j0);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e <= room) sum[e] += ex2(__ldcg(scores + r * P.pitch + e) - x);
            }
        }
    }
    if (STREAM) {
        if (P.S % 4 == 0 && reinterpret_cast<uintptr_t>(P.weights) % 16 == 0 && j0 + 3 < pos) {
            float4* to = reinterpret_cast<float4*>(weights + j0);
            const float4 was = __ldcg(to);
            *to = make_float4(was.x + sum[0], was.y + sum[1], was.z + sum[2], was.w + sum[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (j0 + e < len) weights[j0 + e] = j0 + e < pos ? __ldcg(weights + j0 + e) + sum[e] : sum[e];
        }
        return;
    }
    sm[threadIdx.x] = make_float4(sum[0], sum[1], sum[2], sum[3]);
    __syncthreads();
    const int j = first_key + threadIdx.x;                               // a key each
    if (j >= len) return;
    const float* parts = reinterpret_cast<const float*>(sm) + threadIdx.x;
    float w = 0.f;
#pragma unroll
    for (int k = 0; k < W::GROUPS; ++k) w += parts[k * W::KEYS];
    weights[j] = j < pos ? __ldcg(weights + j) + w : w;
}

// ---------------------------------------------------------------------------------------------------------------- host
constexpr int SMS = 148;

// More than 16 rows of a KV head go to the 5th-generation tensor cores from this many operations (4 D rows keys, by the sizes of the call) on.  mma.sync /
// there, cold caches, 32/8 heads, window 4096: head_dim 128, 5 tokens of 32 sequences (1.1e10) 186 / 120 us, 8 of 8 (4.3e9) 64 / 53, 16 of 4 (4.3e9) 43.0 / 41.0, 40
// of 1 (2.7e9) 36.8 / 34.8, 32 of 1 (2.2e9) 34.8 / 34.8; 64, 32 of 4 (4.3e9) 43.2 / 34.8, 8 of 16 under a window of 2048 (2.2e9) 45 / 41, 16 of 4 (2.2e9) 30.7 /
// 32.8.  Not the scored form: threads that have a row each store its scores piecemeal.
// A prefix whose sequences have such chunks goes there by the same rule (16 tokens of 4 over 8192 rows: 72 / 53).  With few rows each, the prefix there has a launch
// of its own ahead of the own keys, where mma.sync has both in one, so it takes more, counted in pairs of a row and a key, from 32 rows in all on.
// mma.sync / there, 32/8 heads, head_dim 128: 16 sequences over 16384 (8.4e6 pairs) 43 / 49 us, over 32768 (1.7e7) 59 / 64, over 65536 (3.4e7) 94 / 86; 8 over 65536 (1.7e7)
// 88 / 82; 32 over 8192 (8.4e6) beside up to 2000 own keys 82 / 84, over 16384 (1.7e7) 70 / 60; 64 beside 1000 own keys over 4096 (8.4e6) 81 / 86, over 8192 (1.7e7) 94 / 93;
// 128 over 4096 (1.7e7) beside 100 own keys 121 / 62, beside 1000 128 / 113; head_dim 64, 32 over 8192 (8.4e6) 41 / 39, 64 over 6000 (1.2e7) beside 1000 55 / 65, 128 over
// 4096 (1.7e7) beside 1000 86 / 85.
constexpr int TC_TILE = 128, TC_PREFIX_ROWS = 32;           // rows of a tile; rows from which a prefix may go there
constexpr double TC_WORK = 2e9, TC_PREFIX_PAIRS = 1.3e7;
static double work_of(int D, int64_t rows, int64_t items, int64_t keys) { return 4.0 * D * static_cast<double>(rows) * static_cast<double>(items) * static_cast<double>(keys); }
// One launch of clusters, or the stream kernel and the join: as long as a CTA has 16 steps at most and all CTAs run at once.  Captured in a graph,
// 32/8 heads, clusters / stream: head_dim 128, one sequence of 4000 keys 10.3 / 11.3 us, 4 of 2000 10.1 / 14.2, 16 of 1000 13.9 / 18.7, 32 of 1000
// 25.8 / 29.2, 64 of 500 (more CTAs than at once) stays 30.6; head_dim 64, 8 of 1000 8.2 / 13.8.  Clusters of 16 find room in a GPC only where an SM holds
// two of its CTAs, and then one a GPC: 2 sequences of 4000 keys at head_dim 128 took 19.4 us in sixteens, 13.4 streamed; with one CTA an SM, also
// those of 8 only as many as there are GPCs.
constexpr int CLUSTER_MAX = 16, CLUSTER_STEPS = 16, SM_SMEM = 228 * 1024, CLUSTER_SMEM = 225 * 1024;      // (most a CTA may ask for, beside what it has statically)
constexpr size_t cluster_smem(int D) { return D == 64 ? StreamCfg<64>::SMEM : (D == 128 ? StreamCfg<128>::SMEM : StreamCfg<256>::SMEM); }

// CTAs of the kernels for few rows that the GPU holds at once, by their shared memory.
constexpr int resident_ctas(int D) { return SMS * (D == 64 ? 3 : (D == 128 ? 2 : 1)); }

// How a call's work is laid out; a function of its sizes alone, so that the workspace's size is one too.
struct Plan {
    bool stream;                         // few rows: span_stream_kernel
    int cluster, cluster_steps;          // few rows, few steps: span_cluster_kernel with this many CTAs, of this many steps at most
    bool tc, pre_tc;                     // more rows, the own keys / the prefix: span_tc_kernel, not span_rows_kernel
    int ctas, splits, tiles, pre_splits, pre_tiles;
    size_t cum, begun, part_lse, part_o, pre_lse, pre_o, scores, bytes;    // byte offsets in the workspace
    int64_t pitch;
};

static size_t align256(size_t v) { return (v + 255) / 256 * 256; }

// CTAs that share a tile's keys: rounds of resident CTAs times a CTA's steps (and about four steps' time to begin and to end it); joining
// partial results costs `join` steps' time, and a little more with every part.
static int choose_splits(int64_t ctas, int64_t steps, int resident, int join) {
    int best = 1;
    int64_t cost = INT64_MAX;
    for (int s = 1; s <= 64 && s <= steps; ++s) {
        const int64_t c = ((ctas * s + resident - 1) / resident) * ((steps + s - 1) / s + 4) * 8 + (s > 1 ? 8 * join + s : 0);
        if (c < cost) {
            cost = c;
            best = s;
        }
    }
    return best;
}

static Plan plan_of(int B, int H, int KV_H, int D, int n, int S, int window, int sinks, int P, bool scored) {
    Plan p = {};
    if (n == 0) return p;
    const int64_t rows = static_cast<int64_t>(n) * (H / KV_H), items = static_cast<int64_t>(B) * KV_H;
    const int64_t seen = window > 0 && static_cast<int64_t>(window) + sinks + n < S ? static_cast<int64_t>(window) + sinks + n : S;
    p.stream = rows <= 16;
    size_t lse_rows, o_rows;
    int64_t own_steps = 0;
    if (p.stream && P == 0) {
        // as many CTAs a (sequence, KV head) as there are steps for, the GPU holds at once and clusters may have
        const int64_t most = (seen + STEP - 1) / STEP;
        for (int ranks = CLUSTER_MAX; ranks >= 1; ranks /= 2) {
            const int64_t per = (most + ranks - 1) / ranks;
            const size_t smem = cluster_smem(D) + (scored ? rows * per * STEP * 4 : 0);
            const int64_t ctas = static_cast<int64_t>((SM_SMEM - 1) / (smem + 2048));           // of an SM (a little kept by the kernel and by the GPU)
            if (ranks / 2 >= most || per > CLUSTER_STEPS || smem > CLUSTER_SMEM || items * ranks > SMS * ctas) continue;
            if (ranks == 16 && (items > 8 * (ctas - 1) || per > CLUSTER_STEPS / 2)) continue;
            if (ranks == 8 && ctas == 1 && items > 8) continue;
            p.cluster = ranks;
            p.cluster_steps = static_cast<int>(per);
            return p;
        }
    }
    if (p.stream) {
        const int64_t steps = items * ((seen + STEP - 1) / STEP), most = (steps + MIN_STEPS - 1) / MIN_STEPS;
        const int resident = resident_ctas(D);
        p.ctas = static_cast<int>(most < resident ? most : resident);
        own_steps = steps;
        lse_rows = (2 * static_cast<size_t>(p.ctas) + items) * 16;
        o_rows = P > 0 ? lse_rows : 2 * static_cast<size_t>(p.ctas) * 16;
    } else {
        p.tc = !scored && D <= 128 && work_of(D, rows, items, seen) >= TC_WORK;
        const int kt = D == 256 ? 32 : 64, tr = p.tc ? TC_TILE : 64;
        p.tiles = static_cast<int>((rows + tr - 1) / tr);
        const int64_t span = window > 0 && static_cast<int64_t>(window) + sinks + tr < S ? static_cast<int64_t>(window) + sinks + tr : S;
        p.splits = choose_splits(items * p.tiles, (span + kt - 1) / kt, 2 * SMS, scored || P > 0 ? 0 : 6);
        lse_rows = static_cast<size_t>(items) * p.tiles * p.splits * tr;
        o_rows = P > 0 || p.splits > 1 ? lse_rows : 0;
    }
    if (P > 0) {
        p.pre_tc = D <= 128 && rows * B >= TC_PREFIX_ROWS &&
                   (p.stream ? static_cast<double>(rows) * static_cast<double>(items) * P >= TC_PREFIX_PAIRS : work_of(D, rows, items, P) >= TC_WORK);
        const int kt = D == 256 ? 32 : 64, tr = p.pre_tc ? TC_TILE : 64;
        p.pre_tiles = static_cast<int>((rows * B + tr - 1) / tr);
        const int64_t tiles = static_cast<int64_t>(p.pre_tiles) * KV_H, steps = (P + kt - 1) / kt;
        if (p.stream && !p.pre_tc) {
            // one launch: the resident CTAs are shared out by steps, an own step counted half (a cache is seldom full)
            const int64_t resident = resident_ctas(D), share = resident * 2 * steps * tiles / (2 * steps * tiles + own_steps);
            int64_t splits = (share + tiles - 1) / tiles;
            if (splits > (steps + 1) / 2) splits = (steps + 1) / 2;
            p.pre_splits = static_cast<int>(splits < 1 ? 1 : splits);
            const int64_t rest = resident - p.pre_splits * tiles, least = resident / 4;
            if (p.ctas > (rest > least ? rest : least)) p.ctas = static_cast<int>(rest > least ? rest : least);
            lse_rows = o_rows = (2 * static_cast<size_t>(p.ctas) + items) * 16;
        } else {
            p.pre_splits = choose_splits(tiles, steps, 2 * SMS, 0);
        }
    }
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at = align256(at + bytes);
        return here;
    };
    p.cum = take((static_cast<size_t>(B) + 1) * 4);
    p.begun = take(8);
    p.part_lse = take(lse_rows * 4);
    p.part_o = take(o_rows * D * 4);
    if (P > 0) {
        const int tr = p.pre_tc ? TC_TILE : 64;
        const size_t r = static_cast<size_t>(p.pre_tiles) * KV_H * p.pre_splits * tr;
        p.pre_lse = take(r * 4);
        p.pre_o = take(r * D * 4);
    }
    if (scored) {
        p.pitch = (static_cast<int64_t>(S) + 3) / 4 * 4;
        p.scores = take(static_cast<size_t>(items) * rows * p.pitch * 4);
    }
    p.bytes = at;
    return p;
}

// The scored form keeps its scores, 4 bytes a query row and cache row, until their rows' sums are known.  Calls with more than this much of them
// run as several, of as many tokens as fit each: the weights of a token's own row are set by its part and added to by those behind it, as in calls
// one after another.  A token at a time there is nothing left to divide: B * H * S * 4 bytes, G / D of what the cache has.
constexpr int64_t SCORES_MOST = int64_t(1) << 30;
static int scored_tokens(int B, int H, int n, int S) {
    const int64_t token = static_cast<int64_t>(B) * H * ((static_cast<int64_t>(S) + 3) / 4 * 4) * 4;
    const int64_t fit = token < SCORES_MOST ? SCORES_MOST / token : 1;
    if (n <= fit) return n;
    const int64_t parts = (n + fit - 1) / fit;
    return static_cast<int>((n + parts - 1) / parts);
}

// A kernel with more dynamic shared memory than the default, once per device.
template <typename K>
static int allow_smem(K kern, int bytes, bool (&done)[64]) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
    if (!done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) {
            set_cuda_error(e);
            return ALLOYB_E_CUDA;
        }
        done[dev] = true;
    }
    return ALLOYB_OK;
}
template <typename K>
static int launch(K kern, dim3 grid, int threads, int smem, int most_smem, bool (&done)[64], cudaStream_t st, const Params& P) {
    const int rc = allow_smem(kern, most_smem, done);
    if (rc != ALLOYB_OK) return rc;
    const cudaError_t e = launch_pdl(kern, grid, dim3(threads), smem, st, P);
    if (e != cudaSuccess) {
        set_cuda_error(e);
        return ALLOYB_E_CUDA;
    }
    return ALLOYB_OK;
}

template <int D, bool SCORED>
static int launch_cluster(const Plan& plan, const Params& P, cudaStream_t st) {
    static bool ready[64] = {}, wide[64] = {};
    auto kern = span_cluster_kernel<D, SCORED>;
    const int extra = SCORED ? P.n * P.G * plan.cluster_steps * STEP * 4 : 0;
    int rc = allow_smem(kern, CLUSTER_SMEM, ready);
    if (rc != ALLOYB_OK) return rc;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
    if (plan.cluster > 8 && !wide[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) {
            set_cuda_error(e);
            return ALLOYB_E_CUDA;
        }
        wide[dev] = true;
    }
    Params p = P;
    p.splits = plan.cluster;
    p.tiles = plan.cluster_steps;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(plan.cluster, P.B * P.KV_H);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = StreamCfg<D>::SMEM + extra;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = plan.cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) {
        set_cuda_error(e);
        return ALLOYB_E_CUDA;
    }
    return check_launch();
}

template <int D, bool SCORED, bool PREFIX>
static int run_d(const Plan& plan, const Params& P, cudaStream_t st) {
    static bool ready[4][64] = {};
    const int items = P.B * P.KV_H, rows = P.n * P.G;
    int rc = ALLOYB_OK;
    if (!PREFIX && plan.cluster) return launch_cluster<D, SCORED>(plan, P, st);
    constexpr int RUN = RunCfg<D>::SMEM, TILES = RowsCfg<D>::SMEM;
    if (PREFIX) {
        const int ctas = plan.pre_tiles * plan.pre_splits * P.KV_H;
        if (plan.pre_tc) rc = launch_span_tc(P, D, true, dim3(plan.pre_tiles * plan.pre_splits, P.KV_H, 1), st);
        else rc = launch(span_prefix_kernel<D>, dim3(ctas + plan.ctas), WARPS * 32, plan.stream && RUN > TILES ? RUN : TILES, RUN > TILES ? RUN : TILES, ready[0], st, P);
        if (rc == ALLOYB_OK && plan.stream && plan.pre_tc) rc = launch(span_stream_prefix_kernel<D>, dim3(plan.ctas), WARPS * 32, RUN, RUN, ready[3], st, P);
    } else if (plan.stream) {
        rc = launch(span_stream_kernel<D, SCORED>, dim3(plan.ctas), WARPS * 32, RUN, RUN, ready[1], st, P);
    }
    if (rc == ALLOYB_OK && !plan.stream)
        rc = plan.tc ? launch_span_tc(P, D, false, dim3(plan.tiles * plan.splits, P.KV_H, P.B), st)
                     : launch(span_rows_kernel<D, SCORED>, dim3(plan.tiles * plan.splits, P.KV_H, P.B), WARPS * 32, TILES, TILES, ready[2], st, P);
    if (rc != ALLOYB_OK) return rc;
    cudaError_t e = cudaSuccess;
    if (SCORED) {
        const int keys = plan.stream ? Weights<true>::KEYS : Weights<false>::KEYS;
        e = launch_pdl(plan.stream ? span_weights_kernel<true> : span_weights_kernel<false>, dim3((P.S + keys - 1) / keys, items), dim3(256), 0, st, P);
    }
    if (e == cudaSuccess && (plan.stream || plan.splits > 1 || PREFIX)) {                    // (else every output is stored)
        Params M = P;
        // a CTA a row where it has many parts, and the GPU holds all of them at once (16 sequences of 4 heads behind 4096 rows: 4 us sooner); else
        // a warp a row (64 sequences of 8 heads: 12 us sooner)
        const int64_t parts = plan.pre_splits + (plan.stream ? plan.ctas / items + 2 : plan.splits);
        M.merge_team = parts > MERGE_WARPS && static_cast<int64_t>(rows) * items <= 8 * SMS ? MERGE_WARPS : 1;
        auto merge = plan.stream ? span_merge_kernel<D, true, SCORED> : span_merge_kernel<D, false, SCORED>;
        e = launch_pdl(merge, dim3((rows * M.merge_team + MERGE_WARPS - 1) / MERGE_WARPS, items), dim3(MERGE_WARPS * 32), 0, st, M);
    }
    if (e != cudaSuccess) {
        set_cuda_error(e);
        return ALLOYB_E_CUDA;
    }
    return check_launch();
}
template <bool SCORED, bool PREFIX>
static int run(const Plan& plan, const Params& P, int D, cudaStream_t st) {
    switch (D) {
        case 64: return run_d<64, SCORED, PREFIX>(plan, P, st);
        case 128: return run_d<128, SCORED, PREFIX>(plan, P, st);
        default: return run_d<256, SCORED, PREFIX>(plan, P, st);
    }
}

static int sizes_ok(int B, int H, int KV_H, int D, int n, int S) {
    if (B <= 0 || H <= 0 || KV_H <= 0 || H % KV_H || S <= 0 || n < 0 || n > S) return ALLOYB_E_SHAPE;
    if (D != 64 && D != 128 && D != 256) return ALLOYB_E_SHAPE;
    if (B > MAX_BATCH || static_cast<int64_t>(B) * KV_H > 65535 || static_cast<int64_t>(n) * (H / KV_H) * B > (1 << 28)) return ALLOYB_E_LIMIT;
    return ALLOYB_OK;
}

// The arguments that the three entries share, checked and laid out.  new_k null: the cache holds the rows already.
static int fill(Params& P, const void* q, int64_t q_bs, int64_t q_hs, int64_t q_ts, int q_dtype, void* k, void* v, const void* nk, const void* nv,
                int64_t n_bs, int64_t n_hs, int64_t n_ts, const int32_t* pos, int pos_count, void* out, int B, int H, int KV_H, int D, int n, int S,
                float scale) {
    if (!q || !k || !v || !pos || !out || (nk != nullptr) != (nv != nullptr)) return ALLOYB_E_NULL;
    const int rc = sizes_ok(B, H, KV_H, D, n, S);
    if (rc != ALLOYB_OK) return rc;
    // the stride of a dimension of one element says nothing
    if (B == 1) q_bs = n_bs = 0;
    if (H == 1) q_hs = 0;
    if (KV_H == 1) n_hs = 0;
    if (n <= 1) q_ts = n_ts = 0;
    if (pos_count != 1 && pos_count != B) return ALLOYB_E_SHAPE;
    if (q_dtype != ALLOYB_F16 && q_dtype != ALLOYB_BF16) return ALLOYB_E_DTYPE;
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(nk) | reinterpret_cast<uintptr_t>(nv)) % 16 ||
        reinterpret_cast<uintptr_t>(out) % 8 || reinterpret_cast<uintptr_t>(q) % 2 || reinterpret_cast<uintptr_t>(pos) % 4)
        return ALLOYB_E_ALIGN;
    if (nk && ((n_bs | n_hs | n_ts) % 8)) return ALLOYB_E_ALIGN;
    P = Params{};
    P.q = q; P.q_bs = q_bs; P.q_hs = q_hs; P.q_ts = q_ts; P.q_dtype = q_dtype;
    P.q_vec = ((reinterpret_cast<uintptr_t>(q) | (q_bs * 2) | (q_hs * 2) | (q_ts * 2)) & 15) == 0;
    P.k = static_cast<__half*>(k); P.v = static_cast<__half*>(v); P.S = S;
    P.nk = static_cast<const __half*>(nk); P.nv = static_cast<const __half*>(nv);
    P.n_bs = n_bs; P.n_hs = n_hs; P.n_ts = n_ts;
    P.pos = pos; P.pos_count = pos_count; P.out = out;
    P.B = B; P.H = H; P.KV_H = KV_H; P.G = H / KV_H; P.n = P.n_all = n;
    P.scale_log2 = (scale > 0.f ? scale : 1.0f / sqrtf(static_cast<float>(D))) * 1.4426950408889634f;
    return ALLOYB_OK;
}
static int place(Params& P, const Plan& plan, void* workspace, size_t workspace_bytes) {
    if (plan.bytes == 0) return ALLOYB_OK;                               // one launch that needs none
    if (!workspace) return ALLOYB_E_NULL;
    if (reinterpret_cast<uintptr_t>(workspace) % 256) return ALLOYB_E_ALIGN;
    if (workspace_bytes < plan.bytes) return ALLOYB_E_WORKSPACE;
    char* ws = static_cast<char*>(workspace);
    P.cum = reinterpret_cast<int*>(ws + plan.cum);
    static std::atomic<unsigned long long> calls{0};
    P.begun = reinterpret_cast<unsigned long long*>(ws + plan.begun);
    P.call = ++calls * 0x9e3779b97f4a7c15ull;                            // (odd: no two calls alike, and no number that lies about)
    P.part_lse = reinterpret_cast<float*>(ws + plan.part_lse);
    P.part_o = reinterpret_cast<float*>(ws + plan.part_o);
    P.ctas = plan.ctas; P.splits = plan.splits; P.tiles = plan.tiles; P.pre_splits = plan.pre_splits;
    P.tile_rows = plan.tc ? TC_TILE : 64;
    P.pre_tile_rows = plan.pre_tc ? TC_TILE : 64;
    if (plan.pre_splits) {
        P.pre_lse = reinterpret_cast<float*>(ws + plan.pre_lse);
        P.pre_o = reinterpret_cast<float*>(ws + plan.pre_o);
    }
    if (plan.pitch) {
        P.scores = reinterpret_cast<float*>(ws + plan.scores);
        P.pitch = plan.pitch;
    }
    return ALLOYB_OK;
}

}  // namespace sp

// defined in kv_evict.cu
cudaError_t kv_evict_status(int* status, int clear);

}  // namespace alloyb

using namespace alloyb;

extern "C" size_t alloyb_attn_span_workspace_bytes(int B, int H, int KV_H, int D, int n_tokens, int S_max, int window, int sinks, int prefix_len,
                                                   int scored) {
    if (sp::sizes_ok(B, H, KV_H, D, n_tokens, S_max) != ALLOYB_OK || window < 0 || sinks < 0 || prefix_len < 0) return 0;
    if (!scored) return sp::plan_of(B, H, KV_H, D, n_tokens, S_max, window, sinks, prefix_len, false).bytes;
    const int part = sp::scored_tokens(B, H, n_tokens, S_max), rest = part > 0 ? n_tokens % part : 0;
    const size_t most = sp::plan_of(B, H, KV_H, D, part, S_max, window, sinks, prefix_len, true).bytes;
    const size_t last = sp::plan_of(B, H, KV_H, D, rest, S_max, window, sinks, prefix_len, true).bytes;
    return most > last ? most : last;
}

extern "C" int alloyb_attn_window(const void* q, int64_t q_batch_stride, int64_t q_head_stride, int64_t q_tok_stride, int q_dtype, void* k, void* v,
                                  const void* new_k, const void* new_v, int64_t new_batch_stride, int64_t new_head_stride, int64_t new_tok_stride,
                                  const int32_t* pos, int pos_count, void* out, int B, int H, int KV_H, int D, int n_tokens, int S_max, int window,
                                  int sinks, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    sp::Params P;
    int rc = sp::fill(P, q, q_batch_stride, q_head_stride, q_tok_stride, q_dtype, k, v, new_k, new_v, new_batch_stride, new_head_stride, new_tok_stride,
                      pos, pos_count, out, B, H, KV_H, D, n_tokens, S_max, scale);
    if (rc != ALLOYB_OK) return rc;
    if (window < 1 || sinks < 0) return ALLOYB_E_SHAPE;
    P.window = window;
    P.sinks = sinks;
    const sp::Plan plan = sp::plan_of(B, H, KV_H, D, n_tokens, S_max, window, sinks, 0, false);
    rc = sp::place(P, plan, workspace, workspace_bytes);
    if (rc != ALLOYB_OK || n_tokens == 0) return rc;
    return sp::run<false, false>(plan, P, D, as_stream(stream));
}

extern "C" int alloyb_attn_shared_prefix(const void* q, int64_t q_batch_stride, int64_t q_head_stride, int64_t q_tok_stride, int q_dtype,
                                         const void* prefix_k, const void* prefix_v, int64_t prefix_head_stride, int prefix_len, void* k, void* v,
                                         const void* new_k, const void* new_v, int64_t new_batch_stride, int64_t new_head_stride, int64_t new_tok_stride,
                                         const int32_t* pos, int pos_count, void* out, int B, int H, int KV_H, int D, int n_tokens, int S_max,
                                         float scale, void* workspace, size_t workspace_bytes, void* stream) {
    sp::Params P;
    int rc = sp::fill(P, q, q_batch_stride, q_head_stride, q_tok_stride, q_dtype, k, v, new_k, new_v, new_batch_stride, new_head_stride, new_tok_stride,
                      pos, pos_count, out, B, H, KV_H, D, n_tokens, S_max, scale);
    if (rc != ALLOYB_OK) return rc;
    if (prefix_len < 0) return ALLOYB_E_SHAPE;
    if (prefix_len > 0) {
        if (!prefix_k || !prefix_v) return ALLOYB_E_NULL;
        if (KV_H > 1 && prefix_head_stride < static_cast<int64_t>(prefix_len) * D) return ALLOYB_E_SHAPE;
        if ((reinterpret_cast<uintptr_t>(prefix_k) | reinterpret_cast<uintptr_t>(prefix_v)) % 16 || prefix_head_stride % 8) return ALLOYB_E_ALIGN;
    }
    P.pk = static_cast<const __half*>(prefix_k);
    P.pv = static_cast<const __half*>(prefix_v);
    P.p_hs = prefix_head_stride;
    P.P = prefix_len;
    const sp::Plan plan = sp::plan_of(B, H, KV_H, D, n_tokens, S_max, 0, 0, prefix_len, false);
    rc = sp::place(P, plan, workspace, workspace_bytes);
    if (rc != ALLOYB_OK || n_tokens == 0) return rc;
    return prefix_len > 0 ? sp::run<false, true>(plan, P, D, as_stream(stream)) : sp::run<false, false>(plan, P, D, as_stream(stream));
}

extern "C" int alloyb_attn_scored(const void* q, int64_t q_batch_stride, int64_t q_head_stride, int64_t q_tok_stride, int q_dtype, void* k, void* v,
                                  const void* new_k, const void* new_v, int64_t new_batch_stride, int64_t new_head_stride, int64_t new_tok_stride,
                                  const int32_t* pos, int pos_count, float* weights, void* out, int B, int H, int KV_H, int D, int n_tokens, int S_max,
                                  float scale, void* workspace, size_t workspace_bytes, void* stream) {
    sp::Params P;
    int rc = sp::fill(P, q, q_batch_stride, q_head_stride, q_tok_stride, q_dtype, k, v, new_k, new_v, new_batch_stride, new_head_stride, new_tok_stride,
                      pos, pos_count, out, B, H, KV_H, D, n_tokens, S_max, scale);
    if (rc != ALLOYB_OK) return rc;
    if (!weights) return ALLOYB_E_NULL;
    if (reinterpret_cast<uintptr_t>(weights) % 4) return ALLOYB_E_ALIGN;
    P.weights = weights;
    const int part = sp::scored_tokens(B, H, n_tokens, S_max);
    sp::Plan whole = {};                                                     // (checked ahead of the first part's launches)
    whole.bytes = alloyb_attn_span_workspace_bytes(B, H, KV_H, D, n_tokens, S_max, 0, 0, 0, 1);
    sp::Params probe = P;
    rc = sp::place(probe, whole, workspace, workspace_bytes);
    if (rc != ALLOYB_OK) return rc;
    for (int tok0 = 0; tok0 < n_tokens; tok0 += part) {
        sp::Params p = P;
        p.tok0 = tok0;
        p.n = n_tokens - tok0 < part ? n_tokens - tok0 : part;
        p.q = static_cast<const char*>(q) + tok0 * P.q_ts * 2;
        p.out = static_cast<char*>(out) + static_cast<int64_t>(tok0) * H * D * 2;
        if (new_k) {
            p.nk += tok0 * P.n_ts;
            p.nv += tok0 * P.n_ts;
        }
        const sp::Plan plan = sp::plan_of(B, H, KV_H, D, p.n, S_max, 0, 0, 0, true);
        rc = sp::place(p, plan, workspace, workspace_bytes);
        if (rc == ALLOYB_OK) rc = sp::run<true, false>(plan, p, D, as_stream(stream));
        if (rc != ALLOYB_OK) return rc;
    }
    return ALLOYB_OK;
}

extern "C" int alloyb_span_status(int32_t* status_out, int clear) {
    if (!status_out) return ALLOYB_E_NULL;
    int positions = 0, more = 0, lengths = 0;
    cudaError_t e = cudaDeviceSynchronize();
    if (e == cudaSuccess) e = cudaMemcpyFromSymbol(&positions, sp::g_span_status, sizeof(int));
    if (e == cudaSuccess && clear && positions) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(sp::g_span_status, &zero, sizeof(int));
    }
    if (e == cudaSuccess) e = span_tc_status(&more, clear);
    if (e == cudaSuccess) e = kv_evict_status(&lengths, clear);
    if (e != cudaSuccess) {
        set_cuda_error(e);
        return ALLOYB_E_CUDA;
    }
    *status_out = positions | more | lengths << 1;
    return ALLOYB_OK;
}
