// Eviction from an fp16 cache by accumulated attention weight: of every (sequence, KV head)'s rows the first `sinks`, the last `recent` and,
// of those between, the ones of the largest weight stay (ties: the lower position), in their order, at the front of a cache -- another one
// or the same.
//
// evict_select_kernel, a CTA per (sequence, KV head): the weight that the last row to stay has is found digit by digit
// (a histogram of eleven, eleven and ten bits of the weights in an order-preserving integer form), then the positions above it, and as many
// of those equal to it as are wanted, are written in order.  evict_copy_kernel moves the rows.  Bound: HBM, two rows read and written a
// kept position: 128 items of 4096 kept rows of 3000 to 16384 take 98 us, 5.4 TB/s.  Few items go in one launch (evict_one_kernel).
//
// In place a row only moves towards the front: a CTA owns a slice of columns of one (sequence, KV head) and walks the positions in order,
// all of a batch read before any of it is written, so no row is overwritten before it is read: the same 128 items 133 us.
#include "common.cuh"

namespace alloyb {
namespace ev {

static __device__ int g_evict_status = 0;    // sticky: 1 once a length was out of range
constexpr int THREADS = 1024, WARPS = THREADS / 32;
constexpr int BINS = 2 * THREADS;                // eleven bits
constexpr int SMS = 148, SHARE_MOST = 6 * 1024;  // most rows of a CTA that selects and copies: 24 KB of shared memory
constexpr int64_t ONE_ROWS = 150000;             // kept rows in all up to which one launch does both

struct Params {
    const __half *k, *v;                     // (B, KV_H, S, D)
    const float* w;                          // (B, KV_H, S)
    const int32_t* len;
    int len_count;
    __half *k_out, *v_out;                   // (B, KV_H, S_out, D)
    float* w_out;
    int32_t *kept, *new_len;                 // (B, KV_H, keep), (B,)
    int B, KV_H, D, S, S_out, keep, sinks, recent;
    int share;                               // of evict_one_kernel: rows of a CTA
};

__device__ __forceinline__ int length_of(const Params& P, int b, bool tell) {
    const int n = __ldcg(P.len + (P.len_count == 1 ? 0 : b));
    if (n > P.S || n < 0) {
        if (tell) atomicOr(&g_evict_status, 1);
        return 0;
    }
    return n;
}
// Larger weight, larger integer; the zeros are equal, a NaN is below everything.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One digit of the wanted weight, from the counts of its values in hist: the bin in which the count from the top reaches `left` is added to
// `prefix`, and `left` becomes how many are wanted of that bin.  Clears hist for the next digit.  Every thread of the CTA calls it.
__device__ __forceinline__ void take_digit(int* hist, int* warp_sum, int* found, int shift, uint32_t& prefix, int& left) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    const int bin = BINS - 1 - 2 * threadIdx.x, h0 = hist[bin], h1 = hist[bin - 1];      // two neighbouring bins a thread
    hist[bin] = hist[bin - 1] = 0;
    int upto = h0 + h1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    upto += __reduce_add_sync(0xffffffffu, lane < warp ? warp_sum[lane] : 0);
    const int before = upto - h0 - h1;
    if (before < left && upto >= left) {
        const bool upper = before + h0 >= left;
        found[0] = upper ? bin : bin - 1;
        found[1] = left - before - (upper ? 0 : h0);
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(found[0]) << shift;
    left = found[1];
}

constexpr int runs_of(int R) { return R > 0 ? R * WARPS : WARPS; }
template <int R>
struct SelectShared {
    int hist[BINS], warp_sum[WARPS], found[2];
    uint32_t run_sum[runs_of(R)];            // of 32 positions (R == 0: of a warp's): how many above, and equal << 16
    int run_equal[R > 0 ? 1 : WARPS];
};
// put(i, row): the i-th row that stays is `row` (-1: none), for every i below P.keep, by the threads of a CTA; sh.hist is clear.
// R * THREADS weights at most, R of them in a thread's registers: position k * THREADS + thread.  R == 0: any number, read anew in every pass
// (the positions of a warp then lie side by side in the last two).
template <int R, typename Put>
__device__ __forceinline__ void select(const Params& P, SelectShared<R>& sh, int item, int len, const Put& put) {
    int (&hist)[BINS] = sh.hist, (&warp_sum)[WARPS] = sh.warp_sum, (&found)[2] = sh.found;
    auto& run_sum = sh.run_sum;
    auto& run_equal = sh.run_equal;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (len <= P.keep) {
        for (int i = threadIdx.x; i < P.keep; i += THREADS) put(i, i < len ? i : -1);
        return;
    }
    // len > keep >= sinks + recent: the three parts do not meet
    const int first = P.sinks, last = len - P.recent, count = last - first, want = P.keep - P.sinks - P.recent;
    const float* w = P.w + static_cast<int64_t>(item) * P.S + first;
    uint32_t u[R > 0 ? R : 1];
    if (R > 0) {
        float x[R > 0 ? R : 1];
        const float nan = __uint_as_float(0x7fffffffu);
#pragma unroll
        for (int k = 0; k < R; ++k) x[k] = k * THREADS + threadIdx.x < count ? __ldcg(w + k * THREADS + threadIdx.x) : nan;
        // (places past the last count as NaN: below everything, and behind every position that the limit may fall on)
#pragma unroll
        for (int k = 0; k < R; ++k) u[k] = order_of(x[k]);
    }
    for (int i = threadIdx.x; i < P.sinks; i += THREADS) put(i, i);
    for (int i = threadIdx.x; i < P.recent; i += THREADS) put(P.keep - P.recent + i, last + i);
    if (want == 0) return;
    __syncthreads();
    // the integer form of the want-th largest: `prefix` holds the digits found, `left` how many are wanted of those that share them
    uint32_t prefix = 0u;
    int left = want;
    constexpr int SHIFT[3] = {21, 10, 0}, BITS[3] = {11, 11, 10};
#pragma unroll
    for (int digit = 0; digit < 3; ++digit) {
        auto tell = [&](uint32_t x) {
            if (digit == 0 || x >> (SHIFT[digit] + BITS[digit]) == prefix >> (SHIFT[digit] + BITS[digit]))
                atomicAdd(&hist[(x >> SHIFT[digit]) & ((1u << BITS[digit]) - 1u)], 1);
        };
        if (R > 0) {
#pragma unroll
            for (int k = 0; k < R; ++k) {
                if (k * THREADS >= count) break;
                tell(u[k]);
            }
        } else {
#pragma unroll 4
            for (int i = threadIdx.x; i < count; i += THREADS) tell(order_of(__ldcg(w + i)));
        }
        take_digit(hist, warp_sum, found, SHIFT[digit], prefix, left);
    }
    // positions above the limit, and the first `left` of those equal to it
    const uint32_t below = (1u << lane) - 1u;
    if (R > 0) {
#pragma unroll
        for (int k = 0; k < R; ++k) {
            if (k * THREADS >= count) break;
            const uint32_t is_above = __ballot_sync(0xffffffffu, u[k] > prefix), is_equal = __ballot_sync(0xffffffffu, u[k] == prefix);
            if (lane == 0) run_sum[k * WARPS + warp] = __popc(is_above) | __popc(is_equal) << 16;
        }
        __syncthreads();
        // what lies before each run: a thread adds up its run and those of its warp before it, then the warps before
        const int runs = (count + THREADS - 1) / THREADS * WARPS;
        uint32_t own = static_cast<int>(threadIdx.x) < runs ? run_sum[threadIdx.x] : 0u, upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        if (lane == 31) warp_sum[warp] = static_cast<int>(upto);
        __syncthreads();
        upto += __reduce_add_sync(0xffffffffu, lane < warp ? static_cast<uint32_t>(warp_sum[lane]) : 0u);
        if (static_cast<int>(threadIdx.x) < runs) run_sum[threadIdx.x] = upto - own;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < R; ++k) {
            if (k * THREADS >= count) break;
            const uint32_t is_above = __ballot_sync(0xffffffffu, u[k] > prefix), is_equal = __ballot_sync(0xffffffffu, u[k] == prefix);
            const uint32_t before = run_sum[k * WARPS + warp];
            const int a = static_cast<int>(before & 0xffffu) + __popc(is_above & below), e = static_cast<int>(before >> 16) + __popc(is_equal & below);
            if ((is_above >> lane & 1u) || ((is_equal >> lane & 1u) && e < left)) put(P.sinks + a + min(e, left), first + k * THREADS + static_cast<int>(threadIdx.x));
        }
    } else {
        const int run = (count + WARPS * 32 - 1) / (WARPS * 32) * 32, r0 = min(count, warp * run), r1 = min(count, r0 + run);
        int above = 0, equal = 0;
#pragma unroll 4
        for (int i0 = r0; i0 < r1; i0 += 32) {
            const int i = i0 + lane;
            const uint32_t x = i < r1 ? order_of(__ldcg(w + i)) : 0u;
            above += __popc(__ballot_sync(0xffffffffu, i < r1 && x > prefix));
            equal += __popc(__ballot_sync(0xffffffffu, i < r1 && x == prefix));
        }
        if (lane == 0) {
            run_sum[warp] = above;
            run_equal[warp] = equal;
        }
        __syncthreads();
        above = static_cast<int>(__reduce_add_sync(0xffffffffu, lane < warp ? run_sum[lane] : 0u));
        equal = __reduce_add_sync(0xffffffffu, lane < warp ? run_equal[lane] : 0);
#pragma unroll 4
        for (int i0 = r0; i0 < r1; i0 += 32) {
            const int i = i0 + lane;
            const uint32_t x = i < r1 ? order_of(__ldcg(w + i)) : 0u;
            const uint32_t is_above = __ballot_sync(0xffffffffu, i < r1 && x > prefix), is_equal = __ballot_sync(0xffffffffu, i < r1 && x == prefix);
            const int a = above + __popc(is_above & below), e = equal + __popc(is_equal & below);
            if ((is_above >> lane & 1u) || ((is_equal >> lane & 1u) && e < left)) put(P.sinks + a + min(e, left), first + i);
            above += __popc(is_above);
            equal += __popc(is_equal);
        }
    }
}

template <int R>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(const Params P) {
    pdl_launch_dependents();
    __shared__ SelectShared<R> sh;
    const int item = blockIdx.x, b = item / P.KV_H;
    for (int i = threadIdx.x; i < BINS; i += THREADS) sh.hist[i] = 0;
    pdl_wait();
    const int len = length_of(P, b, threadIdx.x == 0 && item == b * P.KV_H);
    int32_t* kept = P.kept + static_cast<int64_t>(item) * P.keep;
    if (threadIdx.x == 0 && item == b * P.KV_H) P.new_len[b] = min(len, P.keep);
    select<R>(P, sh, item, len, [&](int i, int row) { kept[i] = row; });
}

// Few items, another cache: selection and copy in one launch.  Grid (CTAs of an item, items): every CTA of an item selects for itself, on SMs that would
// be idle, and copies its share of the rows, P.share of them, whose places it keeps in shared memory.  One launch / two, cold: 8 items of 2048 of 8000
// rows 16.4 / 18.4 us (calls from Python 17.9 / 20.1), 2 of 500 10.3 / 12.3, 72 of 2048 40.8 / 41.0; 72 of 4096 of 16000 74.1 / 69.7, 8 of 8192 of 32000 42.9 / 38.1.
template <int R>
__global__ void __launch_bounds__(THREADS) evict_one_kernel(const Params P) {
    pdl_launch_dependents();
    extern __shared__ int32_t list[];
    __shared__ SelectShared<R> sh;
    const int item = blockIdx.y, b = item / P.KV_H, row0 = blockIdx.x * P.share, rows = min(P.share, P.keep - row0);
    for (int i = threadIdx.x; i < BINS; i += THREADS) sh.hist[i] = 0;
    pdl_wait();
    const bool tells = threadIdx.x == 0 && blockIdx.x == 0 && item == b * P.KV_H;
    const int len = length_of(P, b, tells);
    if (tells) P.new_len[b] = min(len, P.keep);
    if (rows <= 0) return;                                   // (the last CTAs of an item whose rows the others have)
    select<R>(P, sh, item, len, [&](int i, int row) {
        if (i >= row0 && i < row0 + rows) list[i - row0] = row;
    });
    __syncthreads();
    const int64_t src = static_cast<int64_t>(item) * P.S, dst = static_cast<int64_t>(item) * P.S_out + row0;
    const int half = P.D / 8, shift = P.D == 64 ? 4 : (P.D == 128 ? 5 : 6), pieces = 1 << shift;      // of a row of K, of both
    constexpr int UNROLL = 4;
    for (int i0 = threadIdx.x; i0 < rows * pieces; i0 += THREADS * UNROLL) {
        uint4 x[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int i = i0 + u * THREADS, r = i >> shift, p = i & (pieces - 1);
            if (i < rows * pieces && list[r] >= 0) x[u] = __ldcg(reinterpret_cast<const uint4*>((p < half ? P.k : P.v) + (src + list[r]) * P.D) + (p & (half - 1)));
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int i = i0 + u * THREADS, r = i >> shift, p = i & (pieces - 1);
            if (i < rows * pieces && list[r] >= 0) __stcg(reinterpret_cast<uint4*>((p < half ? P.k_out : P.v_out) + (dst + r) * P.D) + (p & (half - 1)), x[u]);
        }
    }
    for (int i = threadIdx.x; i < rows; i += THREADS) {
        P.kept[static_cast<int64_t>(item) * P.keep + row0 + i] = list[i];
        if (list[i] >= 0) P.w_out[dst + i] = __ldcg(P.w + src + list[i]);
    }
}

// Another cache: every position on its own.  A warp takes UNROLL rounds of 32 pieces of 16 bytes, K's and V's of a position side by side.
constexpr int COPY_THREADS = 256, UNROLL = 8;
template <int D>
struct CopyCfg {
    static constexpr int PIECES = 2 * D / 8, ROWS = COPY_THREADS * UNROLL / PIECES;      // positions of a CTA
};
template <int D>
__global__ void __launch_bounds__(COPY_THREADS) evict_copy_kernel(const Params P) {
    using C = CopyCfg<D>;
    pdl_launch_dependents();
    const int item = blockIdx.y, row0 = blockIdx.x * C::ROWS;
    pdl_wait();
    const int n = min(length_of(P, item / P.KV_H, false), P.keep);
    if (row0 >= n) return;
    const int32_t* kept = P.kept + static_cast<int64_t>(item) * P.keep;
    const int64_t src = static_cast<int64_t>(item) * P.S, dst = static_cast<int64_t>(item) * P.S_out;
    uint4 x[UNROLL];
    int at[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int row = row0 + (u * COPY_THREADS + threadIdx.x) / C::PIECES;
        at[u] = row < n ? __ldcg(kept + row) : -1;
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int p = (u * COPY_THREADS + threadIdx.x) % C::PIECES;
        const __half* from = p < D / 8 ? P.k : P.v;
        if (at[u] >= 0) x[u] = __ldcg(reinterpret_cast<const uint4*>(from + (src + at[u]) * D) + p % (D / 8));
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
        const int i = u * COPY_THREADS + threadIdx.x, row = row0 + i / C::PIECES, p = i % C::PIECES;
        __half* to = p < D / 8 ? P.k_out : P.v_out;
        if (at[u] >= 0) __stcg(reinterpret_cast<uint4*>(to + (dst + row) * D) + p % (D / 8), x[u]);
    }
    for (int i = threadIdx.x; i < C::ROWS && row0 + i < n; i += COPY_THREADS)
        P.w_out[dst + row0 + i] = __ldcg(P.w + src + __ldcg(kept + row0 + i));
}

// The same cache: grid (slices of 32 bytes of K's and of V's columns, and one for the weights; sequences * KV heads).
template <int D>
__global__ void __launch_bounds__(COPY_THREADS) evict_move_kernel(const Params P) {
    constexpr int SLICES = D / 16, HALF = COPY_THREADS / 2;
    pdl_launch_dependents();
    const int item = blockIdx.y, slice = blockIdx.x;
    pdl_wait();
    const int n = min(length_of(P, item / P.KV_H, false), P.keep);
    const int32_t* kept = P.kept + static_cast<int64_t>(item) * P.keep;
    const int64_t src = static_cast<int64_t>(item) * P.S, dst = static_cast<int64_t>(item) * P.S_out;
    if (slice == 2 * SLICES) {
        for (int i0 = 0; i0 < n; i0 += COPY_THREADS * UNROLL) {
            float x[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int i = i0 + u * COPY_THREADS + threadIdx.x;
                if (i < n) x[u] = __ldcg(P.w + src + __ldcg(kept + i));
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int i = i0 + u * COPY_THREADS + threadIdx.x;
                if (i < n) __stcg(P.w_out + dst + i, x[u]);
            }
        }
        return;
    }
    const __half* from = slice < SLICES ? P.k : P.v;
    __half* to = slice < SLICES ? P.k_out : P.v_out;
    const int col = slice % SLICES * 16 + (threadIdx.x & 1) * 8;
    for (int i0 = 0; i0 < n; i0 += HALF * UNROLL) {
        uint4 x[UNROLL];
        int at[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int i = i0 + u * HALF + (threadIdx.x >> 1);
            at[u] = i < n ? __ldcg(kept + i) : -1;
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (at[u] >= 0) x[u] = __ldcg(reinterpret_cast<const uint4*>(from + (src + at[u]) * D + col));
        __syncthreads();                                     // this batch is read before any of it is written
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (at[u] >= 0) __stcg(reinterpret_cast<uint4*>(to + (dst + i0 + u * HALF + (threadIdx.x >> 1)) * D + col), x[u]);
    }
}

template <int D>
static cudaError_t copy(const Params& P, bool in_place, cudaStream_t st) {
    const int items = P.B * P.KV_H;
    if (in_place) return launch_pdl(evict_move_kernel<D>, dim3(2 * (D / 16) + 1, items), dim3(COPY_THREADS), 0, st, P);
    return launch_pdl(evict_copy_kernel<D>, dim3((P.keep + CopyCfg<D>::ROWS - 1) / CopyCfg<D>::ROWS, items), dim3(COPY_THREADS), 0, st, P);
}

}  // namespace ev

cudaError_t kv_evict_status(int* status, int clear) {
    cudaError_t e = cudaMemcpyFromSymbol(status, ev::g_evict_status, sizeof(int));
    if (e == cudaSuccess && clear && *status) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(ev::g_evict_status, &zero, sizeof(int));
    }
    return e;
}

}  // namespace alloyb

using namespace alloyb;

extern "C" int alloyb_kv_evict(const void* k, const void* v, const float* weights, const int32_t* lengths, int lengths_count, void* k_out, void* v_out,
                               float* weights_out, int32_t* kept, int32_t* new_lengths, int B, int KV_H, int D, int S, int S_out, int keep, int sinks,
                               int recent, void* stream) {
    if (!k || !v || !weights || !lengths || !k_out || !v_out || !weights_out || !kept || !new_lengths) return ALLOYB_E_NULL;
    if (B <= 0 || KV_H <= 0 || S <= 0 || S_out <= 0 || keep <= 0 || keep > S_out || sinks < 0 || recent < 0) return ALLOYB_E_SHAPE;
    if (static_cast<int64_t>(sinks) + recent > keep) return ALLOYB_E_SHAPE;
    if (D != 64 && D != 128 && D != 256) return ALLOYB_E_SHAPE;
    if (lengths_count != 1 && lengths_count != B) return ALLOYB_E_SHAPE;
    const int64_t items = static_cast<int64_t>(B) * KV_H;
    if (items > 65535) return ALLOYB_E_LIMIT;
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16)
        return ALLOYB_E_ALIGN;
    // k_out, v_out and weights_out each are their input or lie apart from every input; no output overlaps another, and kept and new_lengths none of the
    // inputs (the CTAs of a sequence read its length while one of them writes the new one)
    struct Span {
        const void* at;
        int64_t bytes;
    };
    const int64_t row = D * 2, rows_in = items * S, rows_out = items * S_out;
    const Span in[4] = {{k, rows_in * row}, {v, rows_in * row}, {weights, rows_in * 4}, {lengths, static_cast<int64_t>(lengths_count) * 4}};
    const Span out[5] = {{k_out, rows_out * row}, {v_out, rows_out * row}, {weights_out, rows_out * 4}, {kept, items * keep * 4}, {new_lengths, static_cast<int64_t>(B) * 4}};
    auto meet = [](const Span& x, const Span& y) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(x.at), b = reinterpret_cast<uintptr_t>(y.at);
        return a < b + y.bytes && b < a + x.bytes;
    };
    bool in_place = false;
    for (int o = 0; o < 5; ++o) {
        for (int i = 0; i < 4; ++i) {
            if (o == i && o < 3 && out[o].at == in[i].at && S_out == S) in_place = true;
            else if (meet(out[o], in[i])) return ALLOYB_E_SHAPE;
        }
        for (int i = 0; i < o; ++i)
            if (meet(out[o], out[i])) return ALLOYB_E_SHAPE;
    }
    ev::Params P;
    P.k = static_cast<const __half*>(k); P.v = static_cast<const __half*>(v); P.w = weights;
    P.len = lengths; P.len_count = lengths_count;
    P.k_out = static_cast<__half*>(k_out); P.v_out = static_cast<__half*>(v_out); P.w_out = weights_out;
    P.kept = kept; P.new_len = new_lengths;
    P.B = B; P.KV_H = KV_H; P.D = D; P.S = S; P.S_out = S_out; P.keep = keep; P.sinks = sinks; P.recent = recent;
    cudaStream_t st = as_stream(stream);
    // as many weights in registers as a cache of S positions can ask for (16384: 22 us from shared memory); past 32 a thread: none
    const int held = S <= 8 * ev::THREADS ? 8 : S <= 16 * ev::THREADS ? 16 : S <= 32 * ev::THREADS ? 32 : 0;
    const int sharers = static_cast<int>(ev::SMS / items);
    P.share = sharers > 1 ? (keep + sharers - 1) / sharers : 0;
    cudaError_t e;
    if (!in_place && sharers > 1 && (held == 8 || held == 16) && items * keep <= ev::ONE_ROWS && P.share <= ev::SHARE_MOST) {
        e = launch_pdl(held == 8 ? ev::evict_one_kernel<8> : ev::evict_one_kernel<16>, dim3(sharers, static_cast<unsigned>(items)), dim3(ev::THREADS), static_cast<size_t>(P.share) * 4, st, P);
    } else {
        auto select = held == 8 ? ev::evict_select_kernel<8> : held == 16 ? ev::evict_select_kernel<16> : held == 32 ? ev::evict_select_kernel<32> : ev::evict_select_kernel<0>;
        e = launch_pdl(select, dim3(static_cast<unsigned>(items)), dim3(ev::THREADS), 0, st, P);
        if (e == cudaSuccess) {
            switch (D) {
                case 64: e = ev::copy<64>(P, in_place, st); break;
                case 128: e = ev::copy<128>(P, in_place, st); break;
                default: e = ev::copy<256>(P, in_place, st); break;
            }
        }
    }
    if (e != cudaSuccess) {
        set_cuda_error(e);
        return ALLOYB_E_CUDA;
    }
    return check_launch();
}
