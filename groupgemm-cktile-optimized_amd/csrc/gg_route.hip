// Top-k router with counts, the sorted row of every (token, slot) pair and the balance loss, and its
// gradients (gg_route, gg_route_backward in include/gg_moe_layer.h).
//
// A token belongs to L lanes, each with V consecutive experts in registers. The largest logits come out
// one per round: the lanes' own maxima, a maximum over the L lanes, and the lowest lane that has it gives
// up its first value of that size, so equal logits go to the lower expert. Logits are compared as
// unsigned numbers of the same order; softmax is taken of the values (max subtracted, float32).
//
// Rows are a stable counting sort. A workgroup takes a chunk of consecutive tokens, lays the experts of
// its pairs out in LDS and ranks 64 pairs at a time: lanes with the same expert find each other with one
// ballot per bit of its number. A chunk's histogram goes to memory, a second launch turns the histograms
// into running sums, a third adds each pair's start. One chunk needs only the first launch. The
// probabilities' sums for the loss follow the same way, chunk by chunk in a fixed order.
#include <algorithm>

#include "gg_layer.h"

namespace gg {
namespace layer {
namespace {

constexpr int kThreads  = 1024, kWaves = kThreads / 64;
constexpr int kMaxPairs = 1024, kMaxTokens = 128, kSegments = kMaxPairs / 64; // of a chunk

struct RouteArgs {
    const void    *logits;
    const uint8_t *mask;
    int           *experts_out, *rows;
    float         *weights, *lse, *loss, *slope;
    int64_t       *counts, *offs;
    int           *hist;  // [chunks][experts + 1]: pairs of each expert, then tokens that take part
    float         *sums;  // [chunks][experts]: sums of probabilities
    int64_t        tokens, stride;
    int            experts, top_k, renormalize, chunk, chunks; // tokens of a chunk
    bool           vec, balance;
};

template <typename T> struct Value;
template <> struct Value<float> {
    static __device__ __forceinline__ float load(const void *p, int64_t i) { return static_cast<const float *>(p)[i]; }
};
template <> struct Value<BF16> {
    static __device__ __forceinline__ float load(const void *p, int64_t i) {
        return __uint_as_float(static_cast<unsigned>(static_cast<const uint16_t *>(p)[i]) << 16);
    }
};
template <> struct Value<F16> {
    static __device__ __forceinline__ float load(const void *p, int64_t i) {
        return static_cast<float>(static_cast<const _Float16 *>(p)[i]);
    }
};

// V values from element i on (i + V inside the row), from 16-byte (8-byte: four 16-bit) pieces.
template <typename T, int V> __device__ __forceinline__ void load_vec(const void *p, int64_t i, float (&v)[V]) {
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const f32x4 w = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + i + j);
#pragma unroll
            for (int q = 0; q < 4; ++q)
                v[j + q] = w[q];
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(p) + i + j);
            T::pair(w[0], v[j], v[j + 1]);
            T::pair(w[1], v[j + 2], v[j + 3]);
        }
    }
}

// The V logits from expert e0 on; -infinity past the last expert.
template <typename T, int V>
__device__ __forceinline__ void load_logits(const void *p, int64_t row, int e0, int experts, bool vec, float (&v)[V]) {
    if (vec && e0 + V <= experts) {
        load_vec<T, V>(p, row + e0, v);
        return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
        v[j] = e0 + j < experts ? Value<T>::load(p, row + e0 + j) : -__builtin_inff();
}

// Unsigned numbers in the order of the floats: NaN largest, the zeros equal, 0 below every one of them.
constexpr unsigned kNoKey = 0, kNegInf = 0x007fffffu;
__device__ __forceinline__ unsigned key_of(float v) {
    const unsigned b = __float_as_uint(v + 0.f); // -0 + 0 = 0
    return v != v ? 0xffffffffu : b ^ (static_cast<int>(b) < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) {
    return __uint_as_float(k ^ (static_cast<int>(k) < 0 ? 0x80000000u : 0xffffffffu)); // NaN: 0x7fffffff, a NaN
}

template <int L> __device__ __forceinline__ unsigned group_max(unsigned v) {
#pragma unroll
    for (int d = L / 2; d > 0; d >>= 1)
        v = max(v, static_cast<unsigned>(__shfl_xor(static_cast<int>(v), d)));
    return v;
}
template <int L> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int d = L / 2; d > 0; d >>= 1)
        v += __shfl_xor(v, d);
    return v;
}

// Exclusive prefix sums over the threads of a workgroup; `scratch` of kWaves entries.
__device__ __forceinline__ int64_t block_prefix(int64_t v, int64_t *scratch, int64_t *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t   s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t o = __shfl_up(s, d);
        s += lane >= d ? o : 0;
    }
    if (lane == 63)
        scratch[wave] = s;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int i = 0; i < kWaves; ++i) {
        before += i < wave ? scratch[i] : 0;
        all += scratch[i];
    }
    *total = all;
    return before + s - v;
}

// The loss from the experts' totals: thread e has expert e's count and sum of probabilities.
__device__ __forceinline__ void write_loss(const RouteArgs &a, int64_t count, int64_t rows, int64_t live, float sum, float *scratch) {
    const int   e = threadIdx.x;
    const float c = rows > 0 && live > 0
                        ? static_cast<float>(count) * static_cast<float>(a.experts) / (static_cast<float>(rows) * static_cast<float>(live))
                        : 0.f;
    if (e < a.experts)
        a.slope[e] = c;
    const float s = wave_sum(e < a.experts ? c * sum : 0.f);
    if ((e & 63) == 0)
        scratch[e >> 6] = s;
    __syncthreads();
    if (e == 0) {
        float l = 0.f;
        for (int i = 0; i < kWaves; ++i)
            l += scratch[i];
        a.loss[0] = l;
    }
}

// One chunk of tokens a workgroup.
template <typename T, int L, int V> __global__ void __launch_bounds__(kThreads) route_kernel(const RouteArgs a) {
    constexpr int kPer = 64 / L, kExperts = L * V; // tokens a wave has at a time
    __shared__ short    sel[kMaxPairs];            // expert of each pair, -1: none
    __shared__ uint16_t seg_hist[kSegments][kExperts];
    __shared__ float    sum_part[kWaves > kPer ? kWaves : kPer][kExperts];
    __shared__ int      live_part[kWaves];
    __shared__ int64_t  scratch[kWaves];
    __shared__ float    fscratch[kWaves];
    const int     tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int     sub = lane & (L - 1), e0 = sub * V, base_lane = lane & ~(L - 1);
    const int64_t first  = static_cast<int64_t>(blockIdx.x) * a.chunk;
    const int     tokens = static_cast<int>(min(static_cast<int64_t>(a.chunk), a.tokens - first));
    const int     pairs  = tokens * a.top_k;

    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
        acc[j] = 0.f;
    int live_here = 0;
    for (int t = wave * kPer + lane / L; t - lane / L < tokens; t += kWaves * kPer) {
        const bool    inside = t < tokens;
        const int64_t token  = first + (inside ? t : 0);
        const bool    wanted = inside && (a.mask == nullptr || a.mask[token] != 0);
        float v[V];
        load_logits<T, V>(a.logits, token * a.stride, e0, a.experts, a.vec, v);
        unsigned key[V];
        unsigned top = kNoKey;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            key[j] = wanted && e0 + j < a.experts ? key_of(v[j]) : kNoKey;
            top    = max(top, key[j]);
        }
        top             = group_max<L>(top);
        const bool live = top > kNegInf;
        // a token with a NaN has a NaN for its maximum, and so for every probability
        const float most = value_of(top);
        float       sum  = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            v[j] = e0 + j < a.experts ? expf(v[j] - most) : 0.f;
            sum += v[j];
        }
        sum             = group_sum<L>(sum);
        const float inv = 1.f / sum;
        if (live) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                acc[j] = fmaf(v[j], inv, acc[j]);
        }
        if (inside && sub == 0) {
            a.lse[token] = live ? most + logf(sum) : -__builtin_inff();
            live_here += live ? 1 : 0;
        }
        // the rounds; lane s % L keeps slot s
        float picked = 0.f, chosen_sum = 0.f;
        for (int s = 0; s < a.top_k; ++s) {
            unsigned own = key[0];
#pragma unroll
            for (int j = 1; j < V; ++j)
                own = max(own, key[j]);
            const unsigned best = group_max<L>(own);
            const uint64_t have = (__ballot(own == best) >> base_lane) & (L == 64 ? ~0ull : (1ull << L) - 1);
            const int      from = __builtin_ctzll(have);
            int            e    = 0;
#pragma unroll
            for (int j = V - 1; j >= 0; --j)
                e = key[j] == best ? j : e;
            if (sub == from) {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    key[j] = j == e ? kNoKey : key[j];
            }
            e = from * V + __shfl(e, base_lane + from);
            const bool  ok = best > kNegInf;
            const float w  = ok ? expf(value_of(best) - most) : 0.f;
            chosen_sum += w;
            if (inside && sub == s % L) {
                sel[t * a.top_k + s]                 = static_cast<short>(ok ? e : -1);
                a.weights[token * a.top_k + s]       = w; // scaled below, by the same lane
                a.experts_out[token * a.top_k + s]   = ok ? e : -1;
            }
        }
        picked = a.renormalize ? 1.f / chosen_sum : inv;
        if (inside)
            for (int s = sub; s < a.top_k; s += L) {
                float *w = a.weights + token * a.top_k + s;
                *w       = live ? *w * picked : 0.f;
            }
    }

    // sums of probabilities and tokens that take part, wave by wave
    if (a.balance) {
#pragma unroll
        for (int d = L; d < 64; d <<= 1)
#pragma unroll
            for (int j = 0; j < V; ++j)
                acc[j] += __shfl_xor(acc[j], d);
        if (lane < L)
#pragma unroll
            for (int j = 0; j < V; ++j)
                sum_part[wave][e0 + j] = acc[j];
    }
    {
        int n = live_here;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1)
            n += __shfl_xor(n, d);
        if (lane == 0)
            live_part[wave] = n;
    }
    for (int i = tid; i < kSegments * kExperts; i += kThreads)
        (&seg_hist[0][0])[i] = 0;
    __syncthreads();

    // rank of each pair among the 64 of its segment, and the segments' histograms
    const int p = tid, seg = wave;
    const int e = p < pairs ? sel[p] : -1;
    int       rank = 0;
    {
        uint64_t same = __ballot(e >= 0);
#pragma unroll
        for (int b = 1; b < kExperts; b <<= 1) {
            const uint64_t set = __ballot((e & b) != 0);
            same &= (e & b) != 0 ? set : ~set;
        }
        if (e >= 0) {
            rank = __builtin_popcountll(same & ((1ull << lane) - 1));
            if (rank == 0)
                seg_hist[seg][e] = static_cast<uint16_t>(__builtin_popcountll(same));
        }
    }
    __syncthreads();
    // running sums over the segments; the chunk's total
    int total = 0;
    if (tid < a.experts) {
        for (int i = 0; i < kSegments; ++i) {
            const int n      = seg_hist[i][tid];
            seg_hist[i][tid] = static_cast<uint16_t>(total);
            total += n;
        }
    }
    __syncthreads();
    if (e >= 0)
        rank += seg_hist[seg][e];
    float sum = 0.f;
    if (a.balance && tid < a.experts)
        for (int i = 0; i < kWaves; ++i)
            sum += sum_part[i][tid];
    int live = 0;
    for (int i = 0; i < kWaves; ++i)
        live += live_part[i];

    const int64_t pair0 = first * a.top_k;
    if (a.chunks > 1) { // finished by the next launches
        if (p < pairs)
            a.rows[pair0 + p] = rank;
        int *hist = a.hist + static_cast<int64_t>(blockIdx.x) * (a.experts + 1);
        if (tid < a.experts) {
            hist[tid] = total;
            if (a.balance)
                a.sums[static_cast<int64_t>(blockIdx.x) * a.experts + tid] = sum;
        }
        if (tid == 0)
            hist[a.experts] = live;
        return;
    }
    int64_t       all;
    const int64_t before = block_prefix(tid < a.experts ? total : 0, scratch, &all);
    if (tid < a.experts) {
        a.counts[tid] = total;
        a.offs[tid]   = before;
    }
    if (tid == 0)
        a.offs[a.experts] = all;
    // sum_part is read: its first row takes the experts' starts
    __syncthreads();
    int *start = reinterpret_cast<int *>(&sum_part[0][0]);
    if (tid < a.experts)
        start[tid] = static_cast<int>(before);
    __syncthreads();
    if (p < pairs)
        a.rows[pair0 + p] = e >= 0 ? start[e] + rank : -1;
    if (a.balance)
        write_loss(a, total, all, live, sum, fscratch);
}

// The chunks' histograms become running sums over the chunks; the totals go to counts and to one more row of
// hist. 64 columns by 16 slices of the chunks a workgroup.
__global__ void __launch_bounds__(kThreads) scan_kernel(const RouteArgs a) {
    __shared__ int part[kWaves][64];
    const int c = threadIdx.x & 63, slice = threadIdx.x >> 6, col = blockIdx.x * 64 + c, cols = a.experts + 1;
    const int per = (a.chunks + kWaves - 1) / kWaves, from = min(slice * per, a.chunks), to = min(from + per, a.chunks);
    int       s   = 0;
    if (col < cols)
        for (int i = from; i < to; ++i)
            s += a.hist[static_cast<int64_t>(i) * cols + col];
    part[slice][c] = s;
    __syncthreads();
    if (col >= cols)
        return;
    int run = 0, all = 0;
    for (int i = 0; i < kWaves; ++i) {
        run += i < slice ? part[i][c] : 0;
        all += part[i][c];
    }
    for (int i = from; i < to; ++i) {
        int      *h = a.hist + static_cast<int64_t>(i) * cols + col;
        const int n = *h;
        *h          = run;
        run += n;
    }
    if (slice == 0) {
        a.hist[static_cast<int64_t>(a.chunks) * cols + col] = all;
        if (col < a.experts)
            a.counts[col] = all;
    }
}

// Every pair's row: its expert's first row, the expert's pairs in earlier chunks, its rank in the chunk. One
// workgroup more for offs and the loss.
__global__ void __launch_bounds__(kThreads) finish_kernel(const RouteArgs a) {
    __shared__ int     start[kThreads];
    __shared__ int64_t scratch[kWaves];
    __shared__ float   fscratch[kWaves];
    const int  tid = threadIdx.x, cols = a.experts + 1;
    const bool last  = static_cast<int>(blockIdx.x) == a.chunks;
    const int  count = tid < a.experts ? a.hist[static_cast<int64_t>(a.chunks) * cols + tid] : 0;
    int64_t       all;
    const int64_t before = block_prefix(count, scratch, &all);
    if (!last) {
        if (tid < a.experts)
            start[tid] = static_cast<int>(before) + a.hist[static_cast<int64_t>(blockIdx.x) * cols + tid];
        __syncthreads();
        const int64_t first  = static_cast<int64_t>(blockIdx.x) * a.chunk;
        const int     tokens = static_cast<int>(min(static_cast<int64_t>(a.chunk), a.tokens - first));
        if (tid < tokens * a.top_k) {
            const int64_t p = first * a.top_k + tid;
            const int     e = a.experts_out[p];
            a.rows[p]       = e >= 0 ? start[e] + a.rows[p] : -1;
        }
        return;
    }
    if (tid < a.experts)
        a.offs[tid] = before;
    if (tid == 0)
        a.offs[a.experts] = all;
    if (a.balance) {
        float sum = 0.f;
        if (tid < a.experts)
            for (int i = 0; i < a.chunks; ++i)
                sum += a.sums[static_cast<int64_t>(i) * a.experts + tid];
        write_loss(a, count, all, a.hist[static_cast<int64_t>(a.chunks) * cols + a.experts], sum, fscratch);
    }
}

// No tokens: counts and offs of zero, a loss of zero.
__global__ void __launch_bounds__(kThreads) empty_kernel(const RouteArgs a) {
    for (int e = threadIdx.x; e <= a.experts; e += kThreads) {
        a.offs[e] = 0;
        if (e < a.experts) {
            a.counts[e] = 0;
            if (a.balance)
                a.slope[e] = 0.f;
        }
    }
    if (threadIdx.x == 0 && a.balance)
        a.loss[0] = 0.f;
}

struct BackArgs {
    const void  *logits;
    const int   *experts_of;
    const float *weights, *lse, *grad_weights, *grad_loss, *slope;
    void        *out;
    int64_t      tokens, stride;
    int          experts, top_k, renormalize;
    bool         vec, vec_out;
};

// dl = p (G - sum p G) (+ the renormalised weights' own softmax over the chosen). The chosen experts' terms
// reach their lanes through an LDS row of the token, which only its own wave touches.
template <typename T, int L, int V> __global__ void __launch_bounds__(256) route_back_kernel(const BackArgs a) {
    constexpr int kPer = 64 / L, kExperts = L * V;
    __shared__ float extra[4 * kPer][kExperts];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane & (L - 1), e0 = sub * V;
    const int mine = wave * kPer + lane / L; // the token's row of LDS
    const float gl = a.grad_loss != nullptr ? a.grad_loss[0] : 0.f;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 4 * kPer;
    for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * 4 * kPer; t0 < a.tokens; t0 += step) {
        const bool    inside = t0 + mine < a.tokens;
        const int64_t t      = inside ? t0 + mine : a.tokens - 1;
        float v[V], g[V];
        load_logits<T, V>(a.logits, t * a.stride, e0, a.experts, a.vec, v);
        const float lse  = a.lse[t];
        const bool  live = lse > -__builtin_inff() || lse != lse;
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            extra[mine][e0 + j] = 0.f;
            v[j]                = live && e0 + j < a.experts ? expf(v[j] - lse) : 0.f;
            g[j]                = a.grad_loss != nullptr && e0 + j < a.experts ? gl * a.slope[e0 + j] : 0.f;
        }
        float inner = 0.f; // sum of w gw over the slots, for renormalised weights
        if (a.grad_weights != nullptr && a.renormalize) {
            for (int s = sub; s < a.top_k; s += L) {
                const int64_t p = t * a.top_k + s;
                if (static_cast<unsigned>(a.experts_of[p]) < static_cast<unsigned>(a.experts))
                    inner = fmaf(a.weights[p], a.grad_weights[p], inner);
            }
            inner = group_sum<L>(inner);
        }
        wave_sync();
        if (a.grad_weights != nullptr)
            for (int s = sub; s < a.top_k; s += L) {
                const int64_t  p = t * a.top_k + s;
                const unsigned e = static_cast<unsigned>(a.experts_of[p]);
                if (live && e < static_cast<unsigned>(a.experts))
                    extra[mine][e] = a.renormalize ? a.weights[p] * (a.grad_weights[p] - inner) : a.grad_weights[p];
            }
        wave_sync();
        float x[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            x[j] = extra[mine][e0 + j];
            if (!a.renormalize) {
                g[j] += x[j];
                x[j] = 0.f;
            }
            dot = fmaf(v[j], g[j], dot);
        }
        dot = group_sum<L>(dot);
#pragma unroll
        for (int j = 0; j < V; ++j)
            x[j] = fmaf(v[j], g[j] - dot, x[j]);
        wave_sync();
        if (!inside)
            continue;
        const int64_t o = t * a.experts + e0;
        if constexpr (std::is_same_v<T, float>) {
            float *out = static_cast<float *>(a.out) + o;
            if (a.vec_out && e0 + V <= a.experts) {
#pragma unroll
                for (int j = 0; j < V; j += 4)
                    *reinterpret_cast<f32x4 *>(out + j) = f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]};
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (e0 + j < a.experts)
                        out[j] = x[j];
            }
        } else {
            uint16_t *out = static_cast<uint16_t *>(a.out) + o;
            if (a.vec_out && e0 + V <= a.experts) {
#pragma unroll
                for (int j = 0; j < V; j += 4)
                    *reinterpret_cast<u32x2 *>(out + j) = u32x2{T::word(x[j], x[j + 1]), T::word(x[j + 2], x[j + 3])};
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (e0 + j < a.experts)
                        out[j] = static_cast<uint16_t>(T::word(x[j], 0.f));
            }
        }
    }
}

// f(L, V) for a number of experts.
template <typename F> int with_lanes(int experts, F f) {
    using std::integral_constant;
#define GG_LANES(l, v)                                                                                                 \
    if (experts <= l * v)                                                                                              \
        return f(integral_constant<int, l>{}, integral_constant<int, v>{});
    GG_LANES(4, 4) GG_LANES(8, 4) GG_LANES(16, 4) GG_LANES(16, 8) GG_LANES(16, 16) GG_LANES(32, 16)
#undef GG_LANES
    return f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

int chunk_tokens(int top_k) { return std::min(kMaxTokens, kMaxPairs / top_k); }

int check_route(int dtype, int64_t tokens, int experts, int top_k, const void *logits, int64_t stride) {
    if (!is16(dtype) && dtype != GG_DTYPE_FP32)
        return fail(GG_ERR_INVALID, "dtype must be GG_DTYPE_BF16, GG_DTYPE_FP16 or GG_DTYPE_FP32");
    if (tokens < 0 || experts < 1 || top_k < 1 || top_k > experts)
        return fail(GG_ERR_INVALID, "tokens must be >= 0, experts >= 1 and top_k in 1 .. experts");
    if (experts > 1024 || top_k > 32 || tokens > INT32_MAX / top_k)
        return fail(GG_ERR_UNSUPPORTED, "experts must be at most 1024, top_k at most 32 and tokens * top_k below 2^31");
    if (tokens > 0 && logits == nullptr)
        return fail(GG_ERR_INVALID, "logits is null");
    if (tokens > 1 && stride < 0)
        return fail(GG_ERR_INVALID, "logits has a negative row stride");
    if (!aligned(logits, dtype == GG_DTYPE_FP32 ? 4 : 2))
        return fail(GG_ERR_UNSUPPORTED, "logits must be aligned to its elements");
    return GG_OK;
}

// Whether rows can be taken in 16-byte pieces.
bool vector_rows(const void *p, int64_t stride, int64_t tokens, int dtype) {
    return aligned(p, 16) && (tokens <= 1 || stride * (dtype == GG_DTYPE_FP32 ? 4 : 2) % 16 == 0);
}

template <typename T> int run_route(const RouteArgs &a, hipStream_t s) {
    int st = with_lanes(a.experts, [&](auto l, auto v) {
        return launch("route", route_kernel<T, l.value, v.value>, a.chunks, kThreads, s, a);
    });
    if (st == GG_OK && a.chunks > 1) {
        st = launch("route", scan_kernel, (a.experts + 1 + 63) / 64, kThreads, s, a);
        if (st == GG_OK)
            st = launch("route", finish_kernel, static_cast<int64_t>(a.chunks) + 1, kThreads, s, a);
    }
    return st;
}

template <typename T> int run_back(const BackArgs &a, hipStream_t s) {
    return with_lanes(a.experts, [&](auto l, auto v) {
        const int64_t per = 4 * (64 / l.value);
        return launch("route_backward", route_back_kernel<T, l.value, v.value>,
                      std::min((a.tokens + per - 1) / per, int64_t(1) << 20), 256, s, a);
    });
}

} // namespace
} // namespace layer
} // namespace gg

using namespace gg::layer;

extern "C" {

size_t gg_route_workspace(int64_t tokens, int experts, int top_k) {
    if (tokens < 1 || experts < 1 || top_k < 1 || top_k > 32)
        return 0;
    const int64_t chunk = chunk_tokens(top_k), chunks = (tokens + chunk - 1) / chunk;
    if (chunks == 1)
        return 0;
    const size_t hist = ((static_cast<size_t>(chunks) + 1) * (experts + 1) * 4 + 15) / 16 * 16;
    return hist + static_cast<size_t>(chunks) * experts * 4;
}

int gg_route(int dtype, int64_t tokens, int experts, int top_k, int renormalize, const void *logits, int64_t stride,
             const uint8_t *mask, int *experts_out, float *weights, int64_t *counts, int64_t *offs, int *rows, float *lse,
             float *loss, float *slope, void *workspace, size_t workspace_bytes, void *stream) {
    g_error[0] = 0;
    if (const int st = check_route(dtype, tokens, experts, top_k, logits, stride))
        return st;
    if (counts == nullptr || offs == nullptr ||
        (tokens > 0 && (experts_out == nullptr || weights == nullptr || rows == nullptr || lse == nullptr)))
        return fail(GG_ERR_INVALID, "experts_out, weights, counts, offs, rows and lse must be device pointers");
    if ((loss == nullptr) != (slope == nullptr))
        return fail(GG_ERR_INVALID, "loss and slope go together");
    const size_t need = gg_route_workspace(tokens, experts, top_k);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
        return fail(GG_ERR_WORKSPACE, "workspace must be 16-byte aligned and of gg_route_workspace(tokens, experts, top_k) bytes");
    RouteArgs a{};
    a.logits      = logits;
    a.mask        = mask;
    a.experts_out = experts_out;
    a.rows        = rows;
    a.weights     = weights;
    a.lse         = lse;
    a.loss        = loss;
    a.slope       = slope;
    a.counts      = counts;
    a.offs        = offs;
    a.tokens      = tokens;
    a.stride      = stride;
    a.experts     = experts;
    a.top_k       = top_k;
    a.renormalize = renormalize;
    a.chunk       = chunk_tokens(top_k);
    a.chunks      = static_cast<int>((tokens + a.chunk - 1) / a.chunk);
    a.hist        = static_cast<int *>(workspace);
    a.sums        = reinterpret_cast<float *>(static_cast<char *>(workspace) +
                                       ((static_cast<size_t>(a.chunks) + 1) * (experts + 1) * 4 + 15) / 16 * 16);
    a.vec         = vector_rows(logits, stride, tokens, dtype);
    a.balance     = loss != nullptr;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (tokens == 0)
        return launch("route", empty_kernel, 1, kThreads, s, a);
    return dtype == GG_DTYPE_FP32   ? run_route<float>(a, s)
           : dtype == GG_DTYPE_BF16 ? run_route<BF16>(a, s)
                                    : run_route<F16>(a, s);
}

int gg_route_backward(int dtype, int64_t tokens, int experts, int top_k, int renormalize, const void *logits,
                      int64_t stride, const int *experts_out, const float *weights, const float *lse,
                      const float *grad_weights, const float *grad_loss, const float *slope, void *grad_logits,
                      void *stream) {
    g_error[0] = 0;
    if (const int st = check_route(dtype, tokens, experts, top_k, logits, stride))
        return st;
    if (tokens == 0)
        return GG_OK;
    if (lse == nullptr || grad_logits == nullptr)
        return fail(GG_ERR_INVALID, "lse and grad_logits must be device pointers");
    if (grad_weights != nullptr && (experts_out == nullptr || weights == nullptr))
        return fail(GG_ERR_INVALID, "grad_weights needs experts_out and weights");
    if ((grad_loss == nullptr) != (slope == nullptr))
        return fail(GG_ERR_INVALID, "grad_loss and slope go together");
    if (!aligned(grad_logits, dtype == GG_DTYPE_FP32 ? 4 : 2))
        return fail(GG_ERR_UNSUPPORTED, "grad_logits must be aligned to its elements");
    BackArgs a{};
    a.logits       = logits;
    a.experts_of   = experts_out;
    a.weights      = weights;
    a.lse          = lse;
    a.grad_weights = grad_weights;
    a.grad_loss    = grad_loss;
    a.slope        = slope;
    a.out          = grad_logits;
    a.tokens       = tokens;
    a.stride       = stride;
    a.experts      = experts;
    a.top_k        = top_k;
    a.renormalize  = renormalize;
    a.vec          = vector_rows(logits, stride, tokens, dtype);
    a.vec_out      = vector_rows(grad_logits, experts, tokens, dtype);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == GG_DTYPE_FP32   ? run_back<float>(a, s)
           : dtype == GG_DTYPE_BF16 ? run_back<BF16>(a, s)
                                    : run_back<F16>(a, s);
}

} // extern "C"
