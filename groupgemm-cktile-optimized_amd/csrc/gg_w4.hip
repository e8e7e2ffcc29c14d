// Grouped products of few rows with 4-bit weights (gg_gemm_w4 in include/gg_moe_layer.h):
// out[m, n] = sum_k x[m, k] s (q[n, k] - z), s and z of each `group` consecutive k.
//
// What bounds it: the packed weights of the groups that have rows, read once. A wave takes NT tiles of 16
// weight rows and every W-th 128 columns of k; a tile's 16 x 128 weights are one 16-byte load per lane, 1 KB in a
// row, and the operand of four 16x16x32 matrix instructions. A nibble becomes a 16-bit float by two bit operations
// on a word for two of them: rotated to the top of the mantissa of 16.0 it is 16 + q, exact in bf16 and fp16. So
// the sum of a scale's k is sum x (16 + q) - (16 + z) sum x, where the second sum comes from matrix instructions
// too, with a constant -24 (-16 and zero points) for weights, once for the NT tiles, and starts the first one.
// The weights are a matrix instruction's columns: a lane has one scale and zero point. Nothing is rounded before
// the float32 sums. The W partial sums are added through LDS.
#include <algorithm>

#include "gg_layer.h"
#include "gg_w4_choice.h"

namespace gg {
namespace layer {
namespace {

typedef __bf16   bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct W4Args {
    const int64_t *lens, *offs;
    const void    *x, *packed, *scales;
    const uint8_t *zeros;
    void          *out;
    int64_t        total_m;
    int            group_num, n, k, n_tiles, k_tiles, groups; // groups: scales along k
};

template <typename T> struct W4Type;
template <> struct W4Type<BF16> {
    static __device__ __forceinline__ float value(unsigned bits) { return __uint_as_float(bits << 16); }
    static constexpr unsigned mask = 0x00780078u, sixteen = 0x41804180u, minus16 = 0xc180c180u, minus24 = 0xc1c0c1c0u;
    static constexpr int      shift = 3; // of q's lowest bit in the half word
    static __device__ __forceinline__ f32x4 mma(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct W4Type<F16> {
    static __device__ __forceinline__ float value(unsigned bits) {
        return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
    }
    static constexpr unsigned mask = 0x03c003c0u, sixteen = 0x4c004c00u, minus16 = 0xcc00cc00u, minus24 = 0xce00ce00u;
    static constexpr int      shift = 6;
    static __device__ __forceinline__ f32x4 mma(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// Eight nibbles of a word as 16 + q: element 2 i from nibble i, 2 i + 1 from nibble i + 4. The two constants come in
// registers of their own (one scalar at most): a shift and one and-or for two nibbles.
struct Bits {
    unsigned mask, sixteen;
};
template <typename T> __device__ __forceinline__ Bits expand_bits() {
    Bits b{W4Type<T>::mask, W4Type<T>::sixteen};
    asm("" : "+v"(b.mask));
    asm("" : "+s"(b.sixteen));
    return b;
}
template <typename T> __device__ __forceinline__ u32x4 expand(unsigned w, const Bits &b) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        constexpr int up    = W4Type<T>::shift;
        const unsigned turned = 4 * i < up ? w << (up - 4 * i) : w >> (4 * i - up);
        r[i]                  = (turned & b.mask) | b.sixteen;
    }
    return r;
}

typedef __amdgpu_buffer_rsrc_t rsrc_t;
__device__ __forceinline__ rsrc_t resource(const void *p, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, bytes, 0x00020000);
}
// Lane offset `v` (checked against the resource), scalar offset `s`.
__device__ __forceinline__ u32x4 load128(rsrc_t r, int v, int s) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, v, s, 0));
}
__device__ __forceinline__ unsigned load16(rsrc_t r, int v, int s) { return __builtin_amdgcn_raw_buffer_load_b16(r, v, s, 0); }
__device__ __forceinline__ unsigned load8(rsrc_t r, int v, int s) { return __builtin_amdgcn_raw_buffer_load_b8(r, v, s, 0); }

// Of one register: rows (16 lanes) 0 0 2 2 and 1 1 3 3; halves 0 0 and 1 1.
__device__ __forceinline__ u32x2 swap16(unsigned v) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return u32x2{r[0], r[1]};
}
__device__ __forceinline__ u32x2 swap32(unsigned v) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return u32x2{r[0], r[1]};
}

// A group's rows, 0 for a length that cannot be right.
__device__ __forceinline__ int length(int64_t len, int64_t total_m) {
    return len < 0 || len > total_m ? 0 : static_cast<int>(len);
}
__device__ __forceinline__ int length_of(const W4Args &a, int g) { return g < a.group_num ? length(a.lens[g], a.total_m) : 0; }
__device__ __forceinline__ int64_t read_lane(int64_t v, int src) { // into scalar registers
    return static_cast<int64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), src))) |
           (static_cast<int64_t>(__builtin_amdgcn_readlane(static_cast<int>(v >> 32), src)) << 32);
}
__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1)
        v += __shfl_xor(v, d);
    return v;
}

// Sums of v over the lanes up to each one.
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned add_dpp(unsigned v) { // v plus another lane's, of rows ROWS
    return v + static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ unsigned wave_scan(unsigned v) {
    v = add_dpp<0x111, 0xf>(v); // the lane 1, 2, 4, 8 before in a row of 16
    v = add_dpp<0x112, 0xf>(v);
    v = add_dpp<0x114, 0xf>(v);
    v = add_dpp<0x118, 0xf>(v);
    v = add_dpp<0x142, 0xa>(v); // a row's last lane to the next row: rows 1 and 3
    return add_dpp<0x143, 0xc>(v); // lane 31 to rows 2 and 3
}

// The `want`-th piece of ROWS rows of the groups: its group (-1: none), the group's rows and the piece's first one. Its
// weights can be asked for before the group's first row is known. A workgroup for each piece, not for each group, because
// one group with more rows than the others would keep its workgroups busy after all else is done: 32 groups of 2 to 25
// rows of 2880 x 2880 51.8 -> 43.6 us, 8 of 12 to 139 rows of 7168 x 2048 47.1 -> 41.
// 64 groups are looked at first, then 256 at a time: 256 groups of which 29 have rows 21.2 -> 19.8 us against 64 at a time.
struct Found {
    int group, rows, m0;
};
template <int ROWS, int N> // N groups a lane, from g0 on
__device__ __forceinline__ bool find_in(const W4Args &a, rsrc_t lens, int g0, unsigned &want, int lane, Found &f) {
    int len[N];
#pragma unroll
    for (int q = 0; q < N; ++q) { // past the last group: 0
        const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(lens, (g0 + lane * N + q) * 8, 0, 0));
        len[q]        = length(static_cast<int64_t>(v[0] | static_cast<uint64_t>(v[1]) << 32), a.total_m);
    }
    unsigned mine = 0;
#pragma unroll
    for (int q = 0; q < N; ++q)
        mine += (static_cast<unsigned>(len[q]) + ROWS - 1) / ROWS;
    const unsigned upto = wave_scan(mine), all = __builtin_amdgcn_readlane(upto, 63);
    if (want >= all) {
        want -= all;
        return false;
    }
    const int src = __builtin_ctzll(__ballot(upto > want));
    want -= __builtin_amdgcn_readlane(upto - mine, src);
    f = {g0 + src * N, __builtin_amdgcn_readlane(len[0], src), 0};
#pragma unroll
    for (int q = 1; q < N; ++q) {
        const unsigned pieces = (static_cast<unsigned>(f.rows) + ROWS - 1) / ROWS;
        if (f.group == g0 + src * N + q - 1 && want >= pieces) {
            want -= pieces;
            f.group = g0 + src * N + q;
            f.rows  = __builtin_amdgcn_readlane(len[q], src);
        }
    }
    f.m0 = static_cast<int>(want) * ROWS;
    return true;
}
template <int ROWS> __device__ __forceinline__ Found find_piece(const W4Args &a, unsigned want, int lane) {
    const rsrc_t lens = resource(a.lens, a.group_num * 8);
    asm volatile("" : "+v"(lane)); // or the offsets made of it stay in registers through the product (5 %)
    Found f{-1, 0, 0};
    if (!find_in<ROWS, 1>(a, lens, 0, want, lane, f))
        for (int g0 = 64; g0 < a.group_num; g0 += 256)
            if (find_in<ROWS, 4>(a, lens, g0, want, lane, f))
                break;
    return f;
}
// Its first row; -1 if its rows do not lie inside [0, total_m).
__device__ __forceinline__ int64_t first_row(const W4Args &a, const Found &f, int lane) {
    int64_t row0 = 0;
    asm volatile("" : "+v"(lane)); // as above
    if (a.offs != nullptr) {
        row0 = read_lane(a.offs[f.group], 0);
    } else {
        row0 = lane < f.group ? length_of(a, lane) : 0;
        for (int g = 64 + lane; g < f.group; g += 64)
            row0 += length_of(a, g);
        row0 = read_lane(wave_sum64(row0), 0);
    }
    return row0 >= 0 && row0 <= a.total_m && f.rows <= a.total_m - row0 ? row0 : -1;
}

// The scales of a tile, and of zero points z 1 + z / 16, in every lane: rows 0 .. N - 1 of 16 lanes hold one each.
template <typename T, int N, bool ZEROS>
__device__ __forceinline__ void spread_scales(unsigned s, unsigned z, float (&scale)[N], float (&point)[N]) {
    unsigned v[4] = {ZEROS ? s | z << 16 : s};
    if constexpr (N > 1) {
        const u32x2 r = swap16(v[0]); // rows 0 0 2 2, 1 1 3 3
        v[0]          = r[0];
        v[1]          = r[1];
    }
    if constexpr (N == 4) {
        const u32x2 a = swap32(v[0]), b = swap32(v[1]);
        v[0]          = a[0];
        v[2]          = a[1];
        v[1]          = b[0];
        v[3]          = b[1];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        scale[i] = W4Type<T>::value(v[i] & 0xffffu);
        point[i] = ZEROS ? fmaf(static_cast<float>(v[i] >> 16), 0.0625f, 1.f) : 1.f;
    }
}

// What both kernels read of weight tile j (of NT) of a group: resources over its weights, scales and zero points.
template <int NT, bool ZEROS> struct Weights {
    rsrc_t w[NT], s[NT], z[NT];
    __device__ __forceinline__ Weights(const W4Args &a, int group, int tile0) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int64_t tile = static_cast<int64_t>(group) * a.n_tiles + min(tile0 + j, a.n_tiles - 1); // past N: the last again
            w[j] = resource(static_cast<const char *>(a.packed) + tile * a.k_tiles * 1024, a.k_tiles * 1024);
            s[j] = resource(static_cast<const char *>(a.scales) + tile * a.groups * 32, a.groups * 32);
            if constexpr (ZEROS)
                z[j] = resource(a.zeros + tile * a.groups * 16, a.groups * 16);
        }
    }
};
template <int NT> struct TileWords {
    u32x4 w[NT];
};
template <int NT> struct TileScales {
    unsigned s[NT], z[NT]; // lanes of row (of 16) quad % kScales: the tile's scale of that number
};
template <int NT, bool ZEROS>
__device__ __forceinline__ void load_words(TileWords<NT> &t, const Weights<NT, ZEROS> &w, int c, int lane) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
        t.w[j] = load128(w.w[j], lane * 16, c * 1024);
}
template <int NT, bool ZEROS, int kScales>
__device__ __forceinline__ void load_scales(TileScales<NT> &t, const Weights<NT, ZEROS> &w, int c, int lane) { // past K: zeros
    const int at = c * kScales + ((lane >> 4) & (kScales - 1));
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        t.s[j] = load16(w.s[j], at * 32 + (lane & 15) * 2, 0);
        if constexpr (ZEROS)
            t.z[j] = load8(w.z[j], at * 16 + (lane & 15), 0);
    }
}

// What a scale's sums start from: base, times 1 + z / 16 of its column with zero points.
template <bool ZEROS> __device__ __forceinline__ f32x4 started(const f32x4 &base, float point) {
    if constexpr (!ZEROS)
        return base;
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        v[r] = base[r] * point;
    return v;
}

// The end of a scale's k: its sums, scaled, into acc. Sums that did not start from base get it here.
template <int MT, int NT, bool ZEROS, bool BASE_FIRST, int N>
__device__ __forceinline__ void scale_sums(f32x4 (&acc)[MT][NT], f32x4 (&sum)[MT][NT], const f32x4 (&base)[MT],
                                           const float (&scale)[NT][N], const float (&point)[NT][N], int q) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if constexpr (!BASE_FIRST)
                    sum[i][j][r] = ZEROS ? fmaf(point[j][q], base[i][r], sum[i][j][r]) : sum[i][j][r] + base[i][r];
                acc[i][j][r] = fmaf(scale[j][q], sum[i][j][r], acc[i][j][r]);
            }
    // here, and not after the tile's last step, where the compiler would gather them with every step's sums alive
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i)
            asm volatile("" : "+v"(acc[i][j]));
}

// Grid: workgroup (piece of 16 rows, block of 16 NT columns), G k of one scale. The W waves share out the 128-column tiles;
// each loads weights, scales and x one tile ahead, into two sets of registers in turn. x comes through a buffer resource
// that ends at the last row, so rows past it read as zeros and cost no traffic. Three workgroups a CU: 168 registers, which
// the compiler passes into accumulation registers, with moves, unless it is told; of the scalar registers the instances with
// zero points reload four a tile from lanes. 16 groups of 8 rows of 4096 x 4096 (k of
// a scale 128): 32.2 us, 4.3 TB/s of packed weights and scales; 32 of 8 rows of 2880 x 2880 (32, zero points) 42.7, 3.7 TB/s.
// Long k comes nearer to the memory's 5.3 TB/s (32 of 8 rows, 2880 x 5632: 55.0 us, 4.9): a call spends 6 to 8 us on the
// launch, the search for its rows, the first loads and the sum over the waves.
template <typename T, int NT, int W, int G, bool ZEROS>
__global__ void __launch_bounds__(W * 64, NT == 4 ? 3 : 2) w4_kernel(const W4Args a) {
    using X = W4Type<T>;
    constexpr int kSteps  = G / 32;  // matrix steps of one scale
    constexpr int kScales = 128 / G; // scales of one tile
    __shared__ f32x4 part[W][NT][64];
    const Bits bits = expand_bits<T>();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int blocks = (a.n_tiles + NT - 1) / NT;
    const int nb     = static_cast<int>(blockIdx.x) % blocks;
    const int slots  = static_cast<int>(gridDim.x) / blocks;
    for (unsigned want = blockIdx.x / blocks;; want += slots) {
        const Found f = find_piece<16>(a, want, lane);
        if (f.group < 0)
            return;
        const int tile0 = nb * NT;
        const Weights<NT, ZEROS> w(a, f.group, tile0);
        TileWords<NT>  words[2]; // of this tile and the next, in turn
        TileScales<NT> scales[2];
        if (wave < a.k_tiles)
            load_words(words[0], w, wave, lane);
        load_scales<NT, ZEROS, kScales>(scales[0], w, wave, lane);
        const int64_t row0 = first_row(a, f, lane);
        if (row0 < 0)
            continue;
        const int m0 = f.m0;
        const rsrc_t xr = resource(static_cast<const uint16_t *>(a.x) + (row0 + m0) * a.k, min(16, f.rows - m0) * a.k * 2);
        const int    xo = col * a.k * 2 + quad * 16;
        struct Operand {
            u32x4 x[4];
        };
        Operand xs[2];
        auto load_x = [&](Operand &o, int c) { // past K: zeros
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                const int k0 = c * 128 + st * 32;
                o.x[st]      = load128(xr, xo | (k0 < a.k ? 0 : static_cast<int>(0x80000000u)), k0 * 2);
            }
        };
        f32x4 acc[1][NT];
#pragma unroll
        for (int j = 0; j < NT; ++j)
            acc[0][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        load_x(xs[0], wave);
        // one tile; PHASE: which of the two buffers is its own (known here, so nothing is moved between them)
        auto tile = [&](auto phase, int c) {
            constexpr int kMine = decltype(phase)::value, kNext = 1 - kMine;
            if (c + W < a.k_tiles)
                load_words(words[kNext], w, c + W, lane);
            load_scales<NT, ZEROS, kScales>(scales[kNext], w, c + W, lane);
            load_x(xs[kNext], c + W);
            float scale[NT][kScales], point[NT][kScales]; // of this lane's column
#pragma unroll
            for (int j = 0; j < NT; ++j)
                spread_scales<T, kScales, ZEROS>(scales[kMine].s[j], scales[kMine].z[j], scale[j], point[j]);
            f32x4 sum[1][NT], base[1];
            const f32x4 zero{0.f, 0.f, 0.f, 0.f};
            constexpr unsigned kMinus = ZEROS ? X::minus16 : X::minus24;
            const u32x4 minus{kMinus, kMinus, kMinus, kMinus};
#pragma unroll
            for (int step = 0; step < 4; ++step) {
                const bool first = step % kSteps == 0;
                if (first) { // -24 (-16) times the scale's share of sum x, in every column: the sums start from it
                    base[0] = zero;
#pragma unroll
                    for (int s2 = step; s2 < step + kSteps; ++s2)
                        base[0] = X::mma(xs[kMine].x[s2], minus, base[0]);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    sum[0][j] = X::mma(xs[kMine].x[step], expand<T>(words[kMine].w[j][step], bits),
                                       first ? started<ZEROS>(base[0], point[j][step / kSteps]) : sum[0][j]);
                if (step % kSteps == kSteps - 1)
                    scale_sums<1, NT, ZEROS, true, kScales>(acc, sum, base, scale, point, step / kSteps);
            }
        };
        for (int c = wave; c < a.k_tiles; c += 2 * W) {
            tile(std::integral_constant<int, 0>{}, c);
            if (c + W < a.k_tiles)
                tile(std::integral_constant<int, 1>{}, c + W);
        }
        // the waves' sums, in their order; each wave stores every W-th of the NT tiles
        __syncthreads(); // the tiles before are read
#pragma unroll
        for (int j = 0; j < NT; ++j)
            part[wave][j][lane] = acc[0][j];
        __syncthreads();
        for (int u = wave; u < NT; u += W) {
            // a sum lies in lane 16 (row / 4) + column, word row % 4; this lane takes row `col`, columns 4 quad ..
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = 0.f;
#pragma unroll
                for (int p = 0; p < W; ++p)
                    v[i] += part[p][u][(col >> 2) * 16 + quad * 4 + i][col & 3];
            }
            const int m = m0 + col, n = (tile0 + u) * 16 + quad * 4;
            if (m < f.rows && n < a.n) // n % 8 == 0: four columns are all there or none
                *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + (row0 + m) * a.n + n) =
                    u32x2{T::word(v[0], v[1]), T::word(v[2], v[3])};
        }
    }
}

// More rows: pieces of 16 MT, each of the four waves with NT tiles of its own, x's rows shared through two LDS buffers of
// one 128-column tile. A row's 16-byte pieces lie at piece ^ row % 16, so the 16 rows that a matrix operand takes at once
// are in different banks. Four workgroups a CU (128 registers) against three: 64 groups of 16 rows of 2048 x 1408 28.9 ->
// 25.1 us, 16 of 48 rows of 4096 x 4096 65.5 -> 57.8, 32 of 12 rows of 2880 x 2880 50.0 -> 49.0; a third set of weights in
// flight takes that back. What bounds it: matrix and vector instructions, which take about as long, hardly overlap.
template <typename T, int MT, int NT, int G, bool ZEROS>
__global__ void __launch_bounds__(256, 4) w4_rows_kernel(const W4Args a) {
    using X = W4Type<T>;
    constexpr int kSteps  = G / 32;
    constexpr int kScales = 128 / G;
    constexpr bool kBaseFirst = kSteps <= 2; // two steps' x are in registers
    constexpr int kTile   = MT * 16 * 256; // bytes of a tile of x
    constexpr int kOut    = MT * 16 * NT * 32; // bytes of a wave's outputs
    __shared__ __attribute__((aligned(16))) unsigned char lds[2 * kTile > 4 * kOut ? 2 * kTile : 4 * kOut];
    const Bits bits = expand_bits<T>();
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int blocks = (a.n_tiles + 4 * NT - 1) / (4 * NT);
    const int nb     = static_cast<int>(blockIdx.x) % blocks;
    const int slots  = static_cast<int>(gridDim.x) / blocks;
    for (unsigned want = blockIdx.x / blocks;; want += slots) {
        const Found f = find_piece<16 * MT>(a, want, lane);
        if (f.group < 0)
            return;
        const int tile0 = (nb * 4 + wave) * NT;
        const Weights<NT, ZEROS> w(a, f.group, tile0);
        TileWords<NT>  words[2];
        TileScales<NT> next_scales;
        load_words(words[0], w, 0, lane);
        load_scales<NT, ZEROS, kScales>(next_scales, w, 0, lane);
        const int64_t row0 = first_row(a, f, lane);
        if (row0 < 0)
            continue;
        const int m0 = f.m0;
        const rsrc_t xr = resource(static_cast<const uint16_t *>(a.x) + (row0 + m0) * a.k, min(16 * MT, f.rows - m0) * a.k * 2);
        // this thread's pieces: row 16 i + tid / 16, piece tid % 16
        const int xrow = tid >> 4, piece = tid & 15;
        u32x4     xin[MT];
        auto load_x = [&](int c) { // past K: zeros
#pragma unroll
            for (int i = 0; i < MT; ++i)
                xin[i] = load128(xr, ((16 * i + xrow) * a.k * 2 + piece * 16) | (c * 128 + piece * 8 < a.k ? 0 : static_cast<int>(0x80000000u)),
                                 c * 256);
        };
        auto store_x = [&](int c) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
                *reinterpret_cast<u32x4 *>(lds + (c & 1) * kTile + (16 * i + xrow) * 256 + ((piece ^ xrow) << 4)) = xin[i];
        };
        f32x4 acc[MT][NT];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        __syncthreads(); // what was in LDS is read
        load_x(0);
        store_x(0);
        __syncthreads();
        // one tile; PHASE as above
        auto tile = [&](auto phase, int c) {
            constexpr int kMine = decltype(phase)::value, kNext = 1 - kMine;
            float scale[NT][kScales], point[NT][kScales];
#pragma unroll
            for (int j = 0; j < NT; ++j)
                spread_scales<T, kScales, ZEROS>(next_scales.s[j], next_scales.z[j], scale[j], point[j]);
            const bool more = c + 1 < a.k_tiles;
            if (more) {
                load_x(c + 1);
                load_scales<NT, ZEROS, kScales>(next_scales, w, c + 1, lane);
                load_words(words[kNext], w, c + 1, lane);
            }
            const unsigned char *xt = lds + (c & 1) * kTile;
            auto read_x = [&](u32x4(&x)[MT], int step) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    x[i] = *reinterpret_cast<const u32x4 *>(xt + (16 * i + col) * 256 + (((step * 4 + quad) ^ col) << 4));
            };
            f32x4 sum[MT][NT], base[MT];
            const f32x4 zero{0.f, 0.f, 0.f, 0.f};
            constexpr unsigned kMinus = ZEROS ? X::minus16 : X::minus24;
            const u32x4 minus{kMinus, kMinus, kMinus, kMinus};
            u32x4 x[2][MT]; // of this step and the next
            // the waves that multiply go before those that load and store: 5 to 10 % (8 groups of 30 rows of 7168 x 2048 20.1
            // -> 18.9 us when this was added)
            __builtin_amdgcn_s_setprio(1);
            read_x(x[0], 0);
#pragma unroll
            for (int step = 0; step < 4; ++step) {
                const bool first = step % kSteps == 0;
                if (step < 3)
                    read_x(x[(step + 1) & 1], step + 1);
                if (!kBaseFirst || first)
#pragma unroll
                    for (int s2 = step; s2 < (kBaseFirst ? step + kSteps : step + 1); ++s2)
#pragma unroll
                        for (int i = 0; i < MT; ++i)
                            base[i] = X::mma(x[s2 & 1][i], minus, first && s2 == step ? zero : base[i]);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const u32x4 wf = expand<T>(words[kMine].w[j][step], bits);
#pragma unroll
                    for (int i = 0; i < MT; ++i)
                        sum[i][j] = X::mma(x[step & 1][i], wf,
                                           !first       ? sum[i][j]
                                           : kBaseFirst ? started<ZEROS>(base[i], point[j][step / kSteps])
                                                        : zero);
                }
                if (step % kSteps == kSteps - 1)
                    scale_sums<MT, NT, ZEROS, kBaseFirst, kScales>(acc, sum, base, scale, point, step / kSteps);
                __builtin_amdgcn_sched_barrier(0); // a step's operands are not fetched earlier than this
            }
            __builtin_amdgcn_s_setprio(0);
            if (more)
                store_x(c + 1);
            __syncthreads();
        };
        for (int c = 0; c < a.k_tiles; c += 2) {
            tile(std::integral_constant<int, 0>{}, c);
            if (c + 1 < a.k_tiles)
                tile(std::integral_constant<int, 1>{}, c + 1);
        }
        // outputs through LDS, a wave's own part: rows of 16 NT columns, stored 16 bytes (8 columns) a lane
        unsigned char *ot = lds + wave * kOut;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    *reinterpret_cast<uint16_t *>(ot + ((16 * i + quad * 4 + r) * NT * 16 + j * 16 + col) * 2) =
                        static_cast<uint16_t>(T::word(acc[i][j][r], 0.f));
        wave_sync();
        for (int u = lane; u < MT * 16 * NT * 2; u += 64) {
            const int m = u / (NT * 2), n8 = u % (NT * 2), n = tile0 * 16 + n8 * 8;
            if (m0 + m < f.rows && n < a.n)
                *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.out) + (row0 + m0 + m) * a.n + n) =
                    *reinterpret_cast<const u32x4 *>(ot + (m * NT * 16 + n8 * 8) * 2);
        }
    }
}

template <typename K> int launch_w4(K kernel, int rows, int columns, int threads, const W4Args &a, hipStream_t s) {
    const int64_t blocks = (static_cast<int64_t>(a.n_tiles) * 16 + columns - 1) / columns;
    // HIP refuses grids of 2^32 threads: past them the pieces are walked in strides
    const int64_t slots = std::min<int64_t>(w4_pieces(a.group_num, a.total_m, rows), (int64_t(1) << 31) / threads / blocks);
    return launch("gemm_w4", kernel, blocks * slots, threads, s, a);
}

// f(k of one scale, zero points or not)
template <typename F> int with_format(const W4Args &a, int group, F f) {
    using std::integral_constant;
    auto zeros = [&](auto g) { return a.zeros != nullptr ? f(g, std::true_type{}) : f(g, std::false_type{}); };
    return group == 128  ? zeros(integral_constant<int, 128>{})
           : group == 64 ? zeros(integral_constant<int, 64>{})
                         : zeros(integral_constant<int, 32>{});
}
template <typename T, int NT, int W> int launch_few(const W4Args &a, int group, hipStream_t s) {
    return with_format(a, group, [&](auto g, auto z) { return launch_w4(w4_kernel<T, NT, W, g.value, z.value>, 16, 16 * NT, 64 * W, a, s); });
}
template <typename T, int MT, int NT> int launch_rows(const W4Args &a, int group, hipStream_t s) {
    return with_format(a, group, [&](auto g, auto z) { return launch_w4(w4_rows_kernel<T, MT, NT, g.value, z.value>, 16 * MT, 64 * NT, 256, a, s); });
}

template <typename T> int run_w4(const W4Args &a, int group, hipStream_t s) {
    switch (w4_choice(a.group_num, a.total_m, a.n)) {
    case W4Choice::kRows:
        return launch_rows<T, 2, 2>(a, group, s);
    case W4Choice::kFew64:
        return launch_few<T, 4, 4>(a, group, s);
    case W4Choice::kFew32:
        return launch_few<T, 2, 8>(a, group, s);
    default:
        return launch_few<T, 1, 8>(a, group, s);
    }
}

} // namespace
} // namespace layer
} // namespace gg

using namespace gg::layer;

extern "C" int gg_gemm_w4(int dtype, int group_num, int64_t total_m, int64_t n, int64_t k, int group,
                          const int64_t *group_lens, const int64_t *group_offs, const void *x, const void *packed,
                          const void *scales, const uint8_t *zeros, void *out, void *stream) {
    g_error[0] = 0;
    if (!is16(dtype))
        return fail(GG_ERR_INVALID, "dtype must be GG_DTYPE_BF16 or GG_DTYPE_FP16");
    if (group_num < 0 || total_m < 0 || n < 0 || k < 1)
        return fail(GG_ERR_INVALID, "group_num, total_m and n must be >= 0 and k >= 1");
    if (group != 32 && group != 64 && group != 128)
        return fail(GG_ERR_UNSUPPORTED, "group must be 32, 64 or 128");
    if (n % 8 != 0 || k % group != 0)
        return fail(GG_ERR_UNSUPPORTED, "N must be a multiple of 8 and K of group");
    if (n > (1 << 21) || k > (1 << 21) || group_num > 8192 || total_m > (1 << 27)) // 256 groups' pieces: in 32 bits
        return fail(GG_ERR_UNSUPPORTED, "N and K must be at most 2097152, groups at most 8192 and rows at most 134217728");
    if (group_num == 0 || total_m == 0 || n == 0)
        return GG_OK;
    if (group_lens == nullptr || x == nullptr || packed == nullptr || scales == nullptr || out == nullptr)
        return fail(GG_ERR_INVALID, "group_lens, x, packed, scales and out must be device pointers");
    if (!aligned(x, 16) || !aligned(packed, 16) || !aligned(scales, 16) || !aligned(out, 16) || !aligned(zeros, 4))
        return fail(GG_ERR_UNSUPPORTED, "x, packed, scales and out must be 16-byte aligned, zeros 4-byte");
    W4Args a{};
    a.lens      = group_lens;
    a.offs      = group_offs;
    a.x         = x;
    a.packed    = packed;
    a.scales    = scales;
    a.zeros     = zeros;
    a.out       = out;
    a.total_m   = total_m;
    a.group_num = group_num;
    a.n         = static_cast<int>(n);
    a.k         = static_cast<int>(k);
    a.n_tiles   = static_cast<int>((n + 15) / 16);
    a.k_tiles   = static_cast<int>((k + 127) / 128);
    a.groups    = static_cast<int>(k / group);
    return dtype == GG_DTYPE_BF16 ? run_w4<BF16>(a, group, static_cast<hipStream_t>(stream))
                                  : run_w4<F16>(a, group, static_cast<hipStream_t>(stream));
}
