// Top-k router with counts, the sorted row of every (token, slot) pair and the balance loss, and its
// gradients (gg_route, gg_route_backward in include/gg_moe_layer.h).
//
// A token belongs to L lanes, each with V consecutive experts in registers. Logits are compared as unsigned numbers of
// the same order. Packed into one word, the number's upper bits and the expert counted backwards (equal logits go to
// the lower expert), each lane sorts its V with a network; then one value per round comes out: the largest of the
// lanes' first ones, whose lane moves up. Where the bits that packing cuts could matter, two are put in order by their
// whole values, and for more the wave takes all again by whole numbers. Softmax is taken of the values (max subtracted, float32).
//
// Rows are a stable counting sort. A workgroup takes a chunk of consecutive tokens, lays the experts of
// its pairs out in LDS and ranks 64 pairs at a time: lanes with the same expert find each other with one
// ballot per bit of its number. A chunk's histogram goes to memory, a second launch turns the histograms
// into running sums, a third adds each pair's start. One chunk needs only the first launch. The
// probabilities' sums for the loss follow the same way, chunk by chunk in a fixed order.
//
// What bounds it: not the bytes (32768 tokens of 256 experts, float32: 7 us at 5.3 TB/s) but vector instructions and the
// steps that wait for each other. Those tokens, top 8 with the loss: 24 us, 17 for the first launch (about 11 of them the
// issue of its 6.7 million vector instructions, the rest loads, barriers and ranks with one workgroup a CU), 4 for the
// second, 3.5 for the third. 33 tokens, one launch: 7.7; one token 5.7. Asking for the next turn's logits ahead
// loses 2 us: the registers are full. Backward 16640 tokens of 32 experts 3.6.
#include <algorithm>

#include "gg_layer.h"

namespace gg {
namespace layer {
namespace {

constexpr int kThreads  = 1024, kWaves = kThreads / 64;
constexpr int kScanless = 32; // chunks whose histograms the last launch adds up itself (of 256: 30 us with the loss where a scan took 26)
constexpr int kMaxPairs = 1024, kMaxTokens = 128, kSegments = kMaxPairs / 64; // of a chunk

struct RouteArgs {
    const void    *logits;
    const uint8_t *mask;
    int           *experts_out, *rows;
    float         *weights, *lse, *loss, *slope;
    int64_t       *counts, *offs;
    int           *hist;  // [chunks + 1][experts + 1]: pairs of each expert, then tokens that take part; then the totals
    float         *sums;  // [chunks + 1][experts]: sums of probabilities, then their totals
    int64_t        tokens, stride;
    int            dtype, experts, top_k, renormalize, chunk, chunks; // chunk: tokens of one
    bool           vec, balance;
};

// Element i of logits of type `dtype`.
__device__ __forceinline__ float load_one(int dtype, const void *p, int64_t i) {
    if (dtype == GG_DTYPE_FP32)
        return static_cast<const float *>(p)[i];
    const unsigned w = static_cast<const uint16_t *>(p)[i];
    float          lo, hi;
    if (dtype == GG_DTYPE_BF16)
        BF16::pair(w, lo, hi);
    else
        F16::pair(w, lo, hi);
    return lo;
}

// The V logits from element `row` + e0 on; -infinity past the last expert. `vec`: rows are 16-byte aligned.
template <int V>
__device__ __forceinline__ void load_logits(int dtype, const void *p, int64_t row, int e0, int experts, bool vec, float (&v)[V]) {
    if (vec && e0 + V <= experts) {
        if (dtype == GG_DTYPE_FP32) {
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                const f32x4 w = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + row + e0 + j);
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    v[j + q] = w[q];
            }
            return;
        }
        const uint16_t *h = static_cast<const uint16_t *>(p) + row + e0;
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(h + j);
            if (dtype == GG_DTYPE_BF16) {
                BF16::pair(w[0], v[j], v[j + 1]);
                BF16::pair(w[1], v[j + 2], v[j + 3]);
            } else {
                F16::pair(w[0], v[j], v[j + 1]);
                F16::pair(w[1], v[j + 2], v[j + 3]);
            }
        }
        return;
    }
    // one by one; past the last expert its value is asked for again, so that no load waits for a branch
    int at[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
        at[j] = min(e0 + j, experts - 1);
    if (dtype == GG_DTYPE_FP32) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            v[j] = static_cast<const float *>(p)[row + at[j]];
    } else {
        unsigned w[V];
#pragma unroll
        for (int j = 0; j < V; ++j)
            w[j] = static_cast<const uint16_t *>(p)[row + at[j]];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            float hi;
            if (dtype == GG_DTYPE_BF16)
                BF16::pair(w[j], v[j], hi);
            else
                F16::pair(w[j], v[j], hi);
        }
    }
#pragma unroll
    for (int j = 0; j < V; ++j)
        v[j] = e0 + j < experts ? v[j] : -__builtin_inff();
}

// Unsigned numbers in the order of the floats: NaN largest, the zeros equal, 0 below every one of them.
constexpr unsigned kNoKey = 0, kNegInf = 0x007fffffu;
__device__ __forceinline__ unsigned key_of(float v) {
    const unsigned b = __float_as_uint(v + 0.f); // -0 + 0 = 0
    return v != v ? 0xffffffffu : b ^ (static_cast<int>(b) < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ unsigned plain_key(float v) { // of no NaN (a positive one is right, too)
    const int b = __float_as_int(v + 0.f);
    return static_cast<unsigned>(b) ^ (static_cast<unsigned>(b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) {
    return __uint_as_float(k ^ (static_cast<int>(k) < 0 ? 0x80000000u : 0xffffffffu)); // NaN: 0x7fffffff, a NaN
}

// exp(x) for x <= 0: the roundings of the product and of the constant make it off by 1.23 |x| 2^-24 at most, v_exp_f32 by
// one unit.
__device__ __forceinline__ float exp_neg(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// Compare-exchanges of a sorting network for N = 4, 8 or 16 values (odd-even merges).
template <int N> struct Network {
    int pairs[N == 4 ? 5 : N == 8 ? 19 : 63][2] = {};
    constexpr Network() {
        int n = 0;
        for (int p = 1; p < N; p *= 2)
            for (int k = p; k >= 1; k /= 2)
                for (int j = k % p; j + k < N; j += 2 * k)
                    for (int i = 0; i < k; ++i)
                        if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                            pairs[n][0] = i + j;
                            pairs[n][1] = i + j + k;
                            ++n;
                        }
    }
};
template <int N> __device__ __forceinline__ void sort_descending(unsigned (&v)[N]) {
    constexpr Network<N> net;
    constexpr int        count = sizeof(net.pairs) / sizeof(net.pairs[0]);
#pragma unroll
    for (int i = 0; i < count; ++i) {
        const unsigned a = v[net.pairs[i][0]], b = v[net.pairs[i][1]];
        v[net.pairs[i][0]] = max(a, b);
        v[net.pairs[i][1]] = min(a, b);
    }
}

// Exclusive prefix sums over the threads of a workgroup; `scratch` of kWaves entries.
__device__ __forceinline__ int block_prefix(int v, int *scratch, int *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int       s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(s, d);
        s += lane >= d ? o : 0;
    }
    if (lane == 63)
        scratch[wave] = s;
    __syncthreads();
    int before = 0, all = 0;
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

// One chunk of tokens a workgroup. KEEP: values of its own that a lane may give (its share of the top_k + 2 largest);
// SLOTS: of the top_k + 2, those that one lane keeps (lane s % L of the token the s-th).
template <int L, int V, int KEEP, int SLOTS> __global__ void __launch_bounds__(kThreads) route_kernel(const RouteArgs a) {
    constexpr int      kPer = 64 / L, kExperts = L * V; // tokens a wave has at a time
    constexpr unsigned kIndex = kExperts - 1;           // low bits of a packed value
    __shared__ short    sel[kMaxPairs];                 // expert of each pair, -1: none
    __shared__ uint16_t seg_hist[kSegments][kExperts];
    __shared__ float    sum_part[kWaves][kExperts];
    __shared__ int      live_part[kWaves], scratch[kWaves];
    __shared__ float    fscratch[kWaves];
    const int     tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int     sub = lane & (L - 1), e0 = sub * V, base_lane = lane & ~(L - 1);
    const int64_t first  = static_cast<int64_t>(blockIdx.x) * a.chunk;
    const int     tokens = static_cast<int>(min(static_cast<int64_t>(a.chunk), a.tokens - first));
    const int     pairs  = tokens * a.top_k, segments = (pairs + 63) / 64;
    unsigned      mask   = ~kIndex; // (in a register: the and-or below has a constant already)
    asm("" : "+v"(mask));
    const unsigned lane_bits = (L - 1 - sub) * V;
    const int      rounds    = a.top_k + (a.dtype == GG_DTYPE_FP32 ? 2 : 0);

    float acc[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
        acc[j] = 0.f;
    int live_here = 0;
    for (int i = tid; i < segments * kExperts; i += kThreads)
        (&seg_hist[0][0])[i] = 0;
    for (int t = wave * kPer + lane / L; t - lane / L < tokens; t += kWaves * kPer) {
        const bool    inside = t < tokens;
        const int64_t token  = first + (inside ? t : 0), row = token * a.stride;
        const bool    wanted = inside && (a.mask == nullptr || a.mask[token] != 0);
        float    v[V];
        unsigned packed[V], top = 0, low = 0;
        load_logits<V>(a.dtype, a.logits, row, e0, a.experts, a.vec, v); // -infinity past the last expert
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const unsigned key = plain_key(v[j]);
            packed[j]          = (key & mask) | (V - 1 - j);
            top                = max(top, key);
            low |= __float_as_uint(v[j]);
        }
        top        = group_max<L>(top);
        low        = group_reduce<L>(low & kIndex, [](unsigned x, unsigned y) { return x | y; });
        float most = value_of(top), sum = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            v[j] = exp_neg(v[j] - most);
            sum += v[j];
        }
        sum       = group_sum<L>(sum);
        bool live = wanted && top > kNegInf;
        // the top_k + 2 largest packed values in order (of 16-bit logits the top_k largest, see below)
        sort_descending(packed);
#pragma unroll
        for (int j = 0; j < KEEP; ++j)
            packed[j] |= lane_bits;
        unsigned pick[SLOTS];
#pragma unroll
        for (int r = 0; r < SLOTS; ++r) {
            pick[r] = 0;
            for (int i = 0; i < L && r * L + i < rounds; ++i) {
                const unsigned best = group_max<L>(packed[0]);
                pick[r]             = sub == i ? best : pick[r];
                const bool mine     = packed[0] == best;
#pragma unroll
                for (int j = 0; j + 1 < KEEP; ++j)
                    packed[j] = mine ? packed[j + 1] : packed[j];
                packed[KEEP - 1] = mine ? 0 : packed[KEEP - 1];
            }
        }
        // Packing cut the values' last bits: their order is right unless two that follow each other agree in the
        // rest (top_k and the first one out among them). 16-bit logits have no such bits. Two such are put in order by
        // their logits below; where there are more in a row the wave takes the values one by one, which takes so long that
        // one token's need is seen in the time of a launch (32768 of 256 experts, where seven in a thousand have two:
        // 27.6 us when those were taken so, 24.1 now; 4096 of 1024, top 32, 42.6 and 32.8). -infinity is never chosen, whatever its place.
        bool doubt = false, tie = false; // tie: this lane's value with the next lane's
        if (__ballot(low != 0) != 0) {
#pragma unroll
            for (int r = 0; r < SLOTS; ++r) {
                const unsigned up   = static_cast<unsigned>(__shfl(static_cast<int>(pick[r]), base_lane + ((sub + 1) & (L - 1))));
                const unsigned over = r + 1 < SLOTS ? static_cast<unsigned>(__shfl(static_cast<int>(pick[r + 1 < SLOTS ? r + 1 : r]), base_lane)) : 0;
                const unsigned next = sub + 1 < L ? up : over;
                tie |= r * L + sub < a.top_k + (SLOTS == 1) && ((pick[r] ^ next) & ~kIndex) == 0 && pick[r] > (kNegInf | kIndex);
            }
            tie &= low != 0;
            if constexpr (SLOTS > 1) {
                doubt = tie;
            } else {
                const uint64_t ties = (__ballot(tie) >> base_lane) & (L == 64 ? ~0ull : (1ull << L) - 1); // of this token
                doubt               = (ties & ties >> 1) != 0;
            }
        }
        // A NaN sum: a NaN, an infinity, or nothing but -infinity. Then too the wave takes the values one by one.
        doubt |= sum != sum;
        int   slot[SLOTS]; // experts
        float x[SLOTS];    // and their logits, -infinity: none
#pragma unroll
        for (int r = 0; r < SLOTS; ++r)
            slot[r] = static_cast<int>(kIndex - (pick[r] & kIndex));
        if (__ballot(doubt && wanted) != 0) {
            unsigned key[V], exact_top = 0;
            float    raw[V];
            load_logits<V>(a.dtype, a.logits, row, e0, a.experts, a.vec, raw);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                key[j]    = e0 + j < a.experts ? key_of(raw[j]) : kNoKey;
                exact_top = max(exact_top, key[j]);
            }
            live = wanted && group_max<L>(exact_top) > kNegInf;
#pragma unroll
            for (int r = 0; r < SLOTS; ++r)
                for (int i = 0; i < L && r * L + i < a.top_k; ++i) {
                    unsigned own = key[0];
#pragma unroll
                    for (int j = 1; j < V; ++j)
                        own = max(own, key[j]);
                    const unsigned best = group_max<L>(own);
                    const uint64_t have = (__ballot(own == best) >> base_lane) & (L == 64 ? ~0ull : (1ull << L) - 1);
                    const int      from = __builtin_ctzll(have); // the lowest lane that has it, its first value of that size
                    int            e    = 0;
#pragma unroll
                    for (int j = V - 1; j >= 0; --j)
                        e = key[j] == best ? j : e;
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        key[j] = sub == from && j == e ? kNoKey : key[j];
                    e       = from * V + __shfl(e, base_lane + from);
                    slot[r] = sub == i ? e : slot[r];
                }
        }
#pragma unroll
        for (int r = 0; r < SLOTS; ++r) {
            x[r] = -__builtin_inff();
            if (live && r * L + sub < a.top_k + (SLOTS == 1) && slot[r] < a.experts)
                x[r] = load_one(a.dtype, a.logits, row + slot[r]);
        }
        if constexpr (SLOTS == 1) {
            const uint64_t firsts = __ballot(tie && !doubt); // (what was taken one by one is in order)
            if (firsts != 0) {
                const bool  first   = (firsts >> lane & 1) != 0, second = sub > 0 && (firsts << 1 >> lane & 1) != 0;
                const int   other   = lane + (first ? 1 : second ? -1 : 0);
                const float x_other = __shfl(x[0], other);
                const int   e_other = __shfl(slot[0], other);
                if (first ? x_other > x[0] : x_other < x[0]) { // equal ones stay: the lower expert is first
                    x[0]    = x_other;
                    slot[0] = e_other;
                }
            }
        }
        float chosen = 0.f;
#pragma unroll
        for (int r = 0; r < SLOTS; ++r)
            chosen += r * L + sub < a.top_k && x[r] != -__builtin_inff() ? exp_neg(x[r] - most) : 0.f;
        const float inv = 1.f / sum, scale = a.renormalize ? 1.f / group_sum<L>(chosen) : inv;
        if (live && a.balance) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                acc[j] = fmaf(v[j], inv, acc[j]);
        }
        if (inside && sub == 0) {
            a.lse[token] = live ? most + logf(sum) : -__builtin_inff();
            live_here += live ? 1 : 0;
        }
#pragma unroll
        for (int r = 0; r < SLOTS; ++r) {
            const int s = r * L + sub;
            if (inside && s < a.top_k) {
                const bool    ok = x[r] != -__builtin_inff(); // -infinity is never chosen
                const int     i  = t * a.top_k + s;
                const int64_t o  = first * a.top_k + i;
                a.weights[o]     = ok ? exp_neg(x[r] - most) * scale : 0.f;
                a.experts_out[o] = ok ? slot[r] : -1;
                sel[i]           = static_cast<short>(ok ? slot[r] : -1);
            }
        }
    }

    // sums of probabilities and tokens that take part, wave by wave
    if (a.balance) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
#pragma unroll
            for (int d = L; d < 16; d <<= 1)
                acc[j] += __shfl_xor(acc[j], d);
            acc[j] = rows_sum<(L > 16 ? L : 16)>(acc[j]);
        }
        if (lane < L)
#pragma unroll
            for (int j = 0; j < V; ++j)
                sum_part[wave][e0 + j] = acc[j];
    }
    {
        const int n = static_cast<int>(group_reduce<64>(static_cast<unsigned>(live_here), [](unsigned x, unsigned y) { return x + y; }));
        if (lane == 0)
            live_part[wave] = n;
    }
    __syncthreads();

    // rank of each pair among the 64 of its segment, and the segments' histograms
    const int p = tid, seg = wave;
    const int e = p < pairs ? sel[p] : -1;
    int       rank = 0;
    if (seg < segments) {
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
    int   total = 0, live = 0;
    float sum   = 0.f;
    if (tid < a.experts) {
        for (int i = 0; i < segments; ++i) {
            const int n      = seg_hist[i][tid];
            seg_hist[i][tid] = static_cast<uint16_t>(total);
            total += n;
        }
        if (a.balance)
            for (int i = 0; i < kWaves; ++i)
                sum += sum_part[i][tid];
    }
    for (int i = 0; i < kWaves; ++i)
        live += live_part[i];
    __syncthreads();
    if (e >= 0)
        rank += seg_hist[seg][e];

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
    int       all;
    const int before = block_prefix(tid < a.experts ? total : 0, scratch, &all);
    int      *start  = reinterpret_cast<int *>(&sum_part[0][0]); // (sum_part is read)
    if (tid < a.experts) {
        a.counts[tid] = total;
        a.offs[tid]   = before;
        start[tid]    = before;
    }
    if (tid == 0)
        a.offs[a.experts] = all;
    __syncthreads();
    if (p < pairs)
        a.rows[pair0 + p] = e >= 0 ? start[e] + rank : -1;
    if (a.balance)
        write_loss(a, total, all, live, sum, fscratch);
}

// The chunks' histograms become running sums over the chunks; the totals go to one more row of hist (and to counts).
// The sums of probabilities: only their totals, to one more row. 16 columns by 64 slices of the chunks a workgroup,
// first the columns of hist, then those of sums. A slice's chunks are loaded kHeld at a time.
template <typename N> __device__ __forceinline__ N slices_before(N s, N (*part)[16], N *total) { // of the 64: in order
    const int c = threadIdx.x & 15, quarter = (threadIdx.x >> 4) & 3, wave = threadIdx.x >> 6;
    const N   one = __shfl_up(s, 16), two = __shfl_up(s, 32), three = __shfl_up(s, 48);
    const N   before = quarter == 0 ? N(0) : quarter == 1 ? one : quarter == 2 ? two + one : three + two + one;
    if (quarter == 3)
        part[wave][c] = before + s;
    __syncthreads();
    N run = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        run += i < wave ? part[i][c] : N(0);
        all += part[i][c];
    }
    *total = all;
    return run + before;
}
__global__ void __launch_bounds__(kThreads) scan_kernel(const RouteArgs a) {
    constexpr int kHeld = 4;
    __shared__ int   part[kWaves][16];
    __shared__ float fpart[kWaves][16];
    const int c = threadIdx.x & 15, slice = threadIdx.x >> 4, cols = a.experts + 1, hist_blocks = (cols + 15) / 16;
    const int per = (a.chunks + 63) / 64, from = min(slice * per, a.chunks), to = min(from + per, a.chunks);
    if (static_cast<int>(blockIdx.x) >= hist_blocks) {
        const int col = min(static_cast<int>((blockIdx.x - hist_blocks) * 16 + c), a.experts - 1); // past the last: it again
        float     s   = 0.f, all;
        for (int i = from; i < to; i += kHeld) {
            float v[kHeld];
#pragma unroll
            for (int j = 0; j < kHeld; ++j)
                v[j] = a.sums[static_cast<int64_t>(min(i + j, to - 1)) * a.experts + col];
#pragma unroll
            for (int j = 0; j < kHeld; ++j)
                s += i + j < to ? v[j] : 0.f;
        }
        slices_before(s, fpart, &all);
        if (slice == 0)
            a.sums[static_cast<int64_t>(a.chunks) * a.experts + col] = all;
        return;
    }
    const int col = min(static_cast<int>(blockIdx.x) * 16 + c, cols - 1);
    const bool mine = static_cast<int>(blockIdx.x) * 16 + c < cols;
    int       v[kHeld], s = 0, all;
    for (int i = from; i < to; i += kHeld) {
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            v[j] = a.hist[static_cast<int64_t>(min(i + j, to - 1)) * cols + col];
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            s += i + j < to ? v[j] : 0;
    }
    int run = slices_before(s, part, &all);
    if (!mine)
        return;
    for (int i = from; i < to; i += kHeld) {
        if (per > kHeld)
#pragma unroll
            for (int j = 0; j < kHeld; ++j)
                v[j] = a.hist[static_cast<int64_t>(min(i + j, to - 1)) * cols + col];
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            if (i + j < to) {
                a.hist[static_cast<int64_t>(i + j) * cols + col] = run;
                run += v[j];
            }
    }
    if (slice == 0) {
        a.hist[static_cast<int64_t>(a.chunks) * cols + col] = all;
        if (col < a.experts)
            a.counts[col] = all;
    }
}

// Every pair's row: its expert's first row, the expert's pairs in earlier chunks, its rank in the chunk. One
// workgroup more for offs and the loss. Of up to kScanless chunks it adds the histograms up itself and there is no
// scan launch.
__global__ void __launch_bounds__(kThreads) finish_kernel(const RouteArgs a) {
    __shared__ int   start[kThreads], scratch[kWaves];
    __shared__ float fscratch[kWaves];
    const int  tid = threadIdx.x, cols = a.experts + 1;
    const bool last   = static_cast<int>(blockIdx.x) == a.chunks;
    const int *totals = a.hist + static_cast<int64_t>(a.chunks) * cols;
    // this workgroup's pairs are asked for before the sums
    const int64_t first = static_cast<int64_t>(blockIdx.x) * a.chunk, p = first * a.top_k + tid;
    const bool    mine  = !last && tid < a.chunk * a.top_k && p < a.tokens * a.top_k;
    const int     e = mine ? a.experts_out[p] : -1, rank = mine ? a.rows[p] : 0;
    int           earlier = 0, count = 0, live = 0, all;
    float         sum = 0.f;
    if (a.chunks <= kScanless) { // the histograms themselves
        if (tid < a.experts) {
#pragma unroll 8
            for (int i = 0; i < a.chunks; ++i) {
                const int n = a.hist[i * cols + tid];
                count += n;
                earlier += i < static_cast<int>(blockIdx.x) ? n : 0;
            }
            if (last && a.balance)
#pragma unroll 8
                for (int i = 0; i < a.chunks; ++i)
                    sum += a.sums[i * a.experts + tid];
        }
        if (last) {
            for (int i = 0; i < a.chunks; ++i)
                live += a.hist[i * cols + a.experts];
            if (tid < a.experts)
                a.counts[tid] = count;
        }
    } else {
        if (tid < a.experts) {
            count   = totals[tid];
            earlier = last ? 0 : a.hist[static_cast<int64_t>(blockIdx.x) * cols + tid];
            sum     = last && a.balance ? a.sums[static_cast<int64_t>(a.chunks) * a.experts + tid] : 0.f;
        }
        live = totals[a.experts];
    }
    const int     before = block_prefix(count, scratch, &all);
    if (!last) {
        if (tid < a.experts)
            start[tid] = before + earlier;
        __syncthreads();
        if (mine)
            a.rows[p] = e >= 0 ? start[e] + rank : -1;
        return;
    }
    if (tid < a.experts)
        a.offs[tid] = before;
    if (tid == 0)
        a.offs[a.experts] = all;
    if (a.balance)
        write_loss(a, count, all, live, sum, fscratch);
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

template <typename T> constexpr int kType = std::is_same_v<T, float> ? int(GG_DTYPE_FP32) : std::is_same_v<T, BF16> ? int(GG_DTYPE_BF16) : int(GG_DTYPE_FP16);

struct BackArgs {
    const void  *logits;
    const int   *experts_of;
    const float *weights, *lse, *grad_weights, *grad_loss, *slope;
    void        *out;
    int64_t      tokens, stride;
    int          experts, top_k, renormalize;
    bool         vec; // rows in and out are 16-byte aligned, so experts come in fours
};

// Four values of logits from element i on.
template <typename T> __device__ __forceinline__ void load_four(const void *p, int64_t i, float &a, float &b, float &c, float &d) {
    if constexpr (std::is_same_v<T, float>) {
        const f32x4 w = *reinterpret_cast<const f32x4 *>(static_cast<const float *>(p) + i);
        a = w[0], b = w[1], c = w[2], d = w[3];
    } else {
        const u32x2 w = *reinterpret_cast<const u32x2 *>(static_cast<const uint16_t *>(p) + i);
        T::pair(w[0], a, b);
        T::pair(w[1], c, d);
    }
}

// dl = p (G - sum p G) (+ the renormalised weights' own softmax over the chosen). The chosen experts' terms
// reach their lanes through an LDS row of the token, which only its own wave touches.
// A lane's value j is that of expert at(j): fours of consecutive ones with VEC, else every L-th, so that a load or store of
// the wave covers consecutive bytes (5219 tokens of 498 experts in float32, a lane's experts consecutive: 26.6 us; so: 10.9).
template <typename T, int L, int V, bool VEC> __global__ void __launch_bounds__(256) route_back_kernel(const BackArgs a) {
    constexpr int kPer = 64 / L, kExperts = L * V;
    __shared__ float extra[4 * kPer][kExperts];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane & (L - 1);
    auto at = [&](int j) { return VEC ? j / 4 * 4 * L + sub * 4 + j % 4 : j * L + sub; };
    const int mine = wave * kPer + lane / L; // the token's row of LDS
    const float gl = a.grad_loss != nullptr ? a.grad_loss[0] : 0.f;
    const int64_t step = static_cast<int64_t>(gridDim.x) * 4 * kPer;
    for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * 4 * kPer; t0 < a.tokens; t0 += step) {
        const bool    inside = t0 + mine < a.tokens;
        const int64_t t      = inside ? t0 + mine : a.tokens - 1;
        float v[V], g[V];
        const int64_t row = t * a.stride;
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < V; j += 4) // (past the last expert: the last four again)
                load_four<T>(a.logits, row + min(at(j), a.experts - 4), v[j], v[j + 1], v[j + 2], v[j + 3]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                v[j] = load_one(kType<T>, a.logits, row + min(at(j), a.experts - 1));
        }
        const float lse  = a.lse[t];
        const bool  live = lse > -__builtin_inff() || lse != lse;
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const bool in      = at(j) < a.experts;
            extra[mine][at(j)] = 0.f;
            v[j]               = live && in ? exp_neg(v[j] - lse) : 0.f;
            g[j]               = a.grad_loss != nullptr && in ? gl * a.slope[at(j)] : 0.f;
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
            x[j] = extra[mine][at(j)];
            if (!a.renormalize) {
                g[j] += x[j];
                x[j] = 0.f;
            }
            dot = fmaf(v[j], g[j], dot);
        }
        dot = group_sum<L>(dot);
#pragma unroll
        for (int j = 0; j < V; ++j)
            x[j] = live ? fmaf(v[j], g[j] - dot, x[j]) : 0.f; // (0 of padding, also where the loss's gradient is infinite)
        wave_sync();
        if (!inside)
            continue;
        const int64_t o = t * a.experts;
        if constexpr (VEC) {
#pragma unroll
            for (int j = 0; j < V; j += 4)
                if (at(j) < a.experts) {
                    if constexpr (std::is_same_v<T, float>)
                        *reinterpret_cast<f32x4 *>(static_cast<float *>(a.out) + o + at(j)) = f32x4{x[j], x[j + 1], x[j + 2], x[j + 3]};
                    else
                        *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + o + at(j)) =
                            u32x2{T::word(x[j], x[j + 1]), T::word(x[j + 2], x[j + 3])};
                }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (at(j) < a.experts) {
                    if constexpr (std::is_same_v<T, float>)
                        static_cast<float *>(a.out)[o + at(j)] = x[j];
                    else
                        static_cast<uint16_t *>(a.out)[o + at(j)] = static_cast<uint16_t>(T::word(x[j], 0.f));
                }
        }
    }
}

// f(L, V) for a number of experts. Of 129 to 256 in the forward pass, 32 lanes of 8 are faster than 16 of 16 while there are few tokens for
// each workgroup, as they take half the time between a turn's loads and its outputs (top 8: 128 tokens 12.7 -> 9.2 us, 4096
// 17.0 -> 14.6, 16384 21.3 -> 20.3; but 33 7.4 -> 7.9, in two turns, and 32768 27.3 -> 28.1, 131072 77 -> 88).
template <typename F> int with_lanes(int experts, bool halves, F f) {
    using std::integral_constant;
#define GG_LANES(l, v)                                                                                                 \
    if (experts <= l * v)                                                                                              \
        return f(integral_constant<int, l>{}, integral_constant<int, v>{});
    GG_LANES(4, 4) GG_LANES(8, 4) GG_LANES(16, 4) GG_LANES(16, 8)
    if (halves) {
        GG_LANES(32, 8)
    }
    GG_LANES(16, 16) GG_LANES(32, 16)
#undef GG_LANES
    return f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
}

bool halves(int64_t tokens) { return tokens > 64 && tokens <= 16384; }

// Tokens of a chunk. All of them where a workgroup takes them in two turns of its waves: one launch. Else a quarter of
// its waves' tokens or more, so that there are about as many chunks as CUs (4096 tokens of 256 experts, top 8: 16 tokens a
// chunk instead of 128).
int chunk_tokens(int64_t tokens, int experts, int top_k) {
    const int most = std::min(kMaxTokens, kMaxPairs / top_k);
    const int turn = with_lanes(experts, halves(tokens), [](auto l, auto) { return kWaves * 64 / l.value; }); // tokens of a workgroup's waves at a time
    if (tokens <= std::min(most, 2 * turn))
        return most;
    const int64_t even = (tokens + 255) / 256, quarter = turn / 4;
    return static_cast<int>(std::min<int64_t>(most, (even + quarter - 1) / quarter * quarter));
}

int check_route(int dtype, int64_t tokens, int experts, int top_k, const void *logits, int64_t stride) {
    if (!is16(dtype) && dtype != GG_DTYPE_FP32)
        return fail(GG_ERR_INVALID, "dtype must be GG_DTYPE_BF16, GG_DTYPE_FP16 or GG_DTYPE_FP32");
    if (tokens < 0 || experts < 1 || top_k < 1 || top_k > experts)
        return fail(GG_ERR_INVALID, "tokens must be >= 0, experts >= 1 and top_k in 1 .. experts");
    if (experts > 1024 || top_k > 32 || tokens > INT32_MAX / top_k)
        return fail(GG_ERR_UNSUPPORTED, "experts must be at most 1024, top_k at most 32 and tokens * top_k below 2^31");
    if (tokens > 1 << 28) // HIP refuses grids of 2^32 threads: 1024 for each chunk of 128 tokens
        return fail(GG_ERR_UNSUPPORTED, "tokens must be at most 268435456");
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

int run_route(const RouteArgs &a, hipStream_t s) {
    int st = with_lanes(a.experts, halves(a.tokens), [&](auto l, auto v) {
        constexpr int few = v.value < 10 ? v.value : 10; // of top_k + 2 <= 10 values
        constexpr int most = l.value * v.value < 32 ? l.value * v.value + 2 : 34; // top_k + 2
        return a.top_k <= 8
                   ? launch("route", route_kernel<l.value, v.value, few, (10 + l.value - 1) / l.value>, a.chunks, kThreads, s, a)
                   : launch("route", route_kernel<l.value, v.value, v.value, (most + l.value - 1) / l.value>, a.chunks, kThreads, s, a);
    });
    if (st == GG_OK && a.chunks > 1) {
        if (a.chunks > kScanless)
            st = launch("route", scan_kernel, (a.experts + 16) / 16 + (a.balance ? (a.experts + 15) / 16 : 0), kThreads, s, a);
        if (st == GG_OK)
            st = launch("route", finish_kernel, static_cast<int64_t>(a.chunks) + 1, kThreads, s, a);
    }
    return st;
}

template <typename T> int run_back(const BackArgs &a, hipStream_t s) {
    return with_lanes(a.experts, false, [&](auto l, auto v) {
        const int64_t per = 4 * (64 / l.value);
        return launch("route_backward", a.vec ? route_back_kernel<T, l.value, v.value, true> : route_back_kernel<T, l.value, v.value, false>,
                      std::min((a.tokens + per - 1) / per, int64_t(1) << 20), 256, s, a);
    });
}

} // namespace
} // namespace layer
} // namespace gg

using namespace gg::layer;

extern "C" {

size_t gg_route_workspace(int64_t tokens, int experts, int top_k) {
    if (tokens < 1 || experts < 1 || experts > 1024 || top_k < 1 || top_k > 32)
        return 0;
    const int64_t chunk = chunk_tokens(tokens, experts, top_k), chunks = (tokens + chunk - 1) / chunk;
    if (chunks == 1)
        return 0;
    const size_t hist = ((static_cast<size_t>(chunks) + 1) * (experts + 1) * 4 + 15) / 16 * 16;
    return hist + (static_cast<size_t>(chunks) + 1) * experts * 4;
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
    a.dtype       = dtype;
    a.experts     = experts;
    a.top_k       = top_k;
    a.renormalize = renormalize;
    a.chunk       = chunk_tokens(tokens, experts, top_k);
    a.chunks      = static_cast<int>((tokens + a.chunk - 1) / a.chunk);
    a.hist        = static_cast<int *>(workspace);
    a.sums        = reinterpret_cast<float *>(static_cast<char *>(workspace) +
                                       ((static_cast<size_t>(a.chunks) + 1) * (experts + 1) * 4 + 15) / 16 * 16);
    a.vec         = vector_rows(logits, stride, tokens, dtype);
    a.balance     = loss != nullptr;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (tokens == 0)
        return launch("route", empty_kernel, 1, kThreads, s, a);
    return run_route(a, s);
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
    // (one token: its experts in fours, too)
    a.vec          = vector_rows(logits, stride, tokens, dtype) && vector_rows(grad_logits, experts, 2, dtype);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == GG_DTYPE_FP32   ? run_back<float>(a, s)
           : dtype == GG_DTYPE_BF16 ? run_back<BF16>(a, s)
                                    : run_back<F16>(a, s);
}

} // extern "C"
