// Attention of one new token of each sequence over a paged cache.
//
// What bounds it is reading the keys and values once; a token's 4*dim*group
// operations are few.  Everything else is arranged so that a wave only loads
// and multiplies:
//
//  - The query heads of a kv head are the 16 columns of the matrix cores'
//    tiles, so keys and values are read once for up to 16 of them (32 where two
//    tiles fit the registers).  Scores are
//    made transposed, S^T = K Q^T (16 keys x 16 heads): a lane then holds, for
//    one head, the scores of keys 4g..4g+3 of each tile (g = lane / 16), and
//    that is just how the second product O^T = V^T P^T wants its right operand
//    if its inner index runs over the keys in the order (tile, g, 0..3).  So
//    weights never leave the lane that made them, softmax needs a lane's own
//    values and two exchanges for the maximum, and no LDS is touched before the
//    waves' sums are joined.
//  - V^T wants eight keys of one column in a lane.  A lane loads neighbouring
//    columns of eight keys (a row of the cache by 16 lanes, all of a page's
//    bytes by a few instructions) and transposes pairs with byte permutes;
//    which columns share a tile does not matter, as each tile's results are
//    written where its columns belong.
//  - 4-bit values are converted in registers (the hardware's conversion with a
//    power-of-two scale, exact in bf16 and in f16 down to its smallest step).
//  - Weights are 2^(score - reference), any reference that keeps them in range.
//    It is raised only when a score comes to lie too far above it, so most steps
//    skip the exchange and the rescaling (Below, Slack).
//  - Weights enter the second product as two values of the 16-bit type, the
//    rounded weight and the rounding's remainder, 16 or more bits together:
//    one alone would make the weights' rounding as large as the output's own.
//    f16's are so small that they are multiplied with the values apart (kRest).
//
// The work is all tokens of all kv heads behind each other, in units of 128 keys,
// and every workgroup that the card holds at once takes an equal share of it:
// the lengths, which only the GPU knows, decide how many workgroups a sequence
// gets.  A share that ends inside a sequence leaves a part; a second launch joins
// the parts, and adds the weights to the tokens' mass where that is tracked.
//
// Measured: 16 sequences of up to 32768 tokens, 40 query heads over 8 of 128
// columns: 269 us in bf16 (1.61 GB, 6.0 TB/s; VALU 10% busy, matrix cores 6%), 85
// us from 4 bits (0.43 GB, 5.0 TB/s; 50% and 21%), and 5 us to join.  A kernel that
// only reads reaches 5.9 to 6.1 TB/s over 2 to 4 GiB.  Short calls are latency: one
// sequence of 32768 tokens over 2 heads 11.5 and 4.0 us, of 5 tokens 5.5 and 2.1.
#include "kv_device.h"

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kUnit = 128;        // keys that work is dealt in: a step of every wave
constexpr int kCus = 256;         // of an MI355X that is not partitioned
constexpr float kLog2e = 1.4426950408889634f;

// The reference is set this far below the largest score so far, and again when
// a score exceeds it by Slack (both log2).  f16 weights begin at 2^13: its smallest
// step is 2^-24, and the largest value 2^16.
template <typename T>
constexpr float kBelow = std::is_same_v<T, _Float16> ? 13.f : 0.f;
template <typename T>
constexpr float kSlack = std::is_same_v<T, _Float16> ? 15.f : 8.f;
// What f16 remainders are multiplied by, so that weights keep 16 bits down to 2^-33
// of the largest.  As they are they do down to 2^-22, and outputs of columns where
// the heavy tokens' values are zero were off by up to six times their rounding; it
// costs 0 to 2% over plain pages and 1 to 4% over 4-bit ones.
template <typename T>
constexpr float kRest = std::is_same_v<T, _Float16> ? 2048.f : 1.f;

struct Attend {
    vramc_kv_cache c;
    const void* q;
    int64_t q_seq, q_head;
    bool q_wide;             // rows of q can be read 16 bytes at a time
    int q_heads, group;
    const int32_t* table;
    int64_t table_row;
    const int32_t* lengths;
    int batch;
    float scale;
    void* out;
    int tile;                // query heads that are taken at once, 16 or 32
    int head_tiles, groups;  // tiles of a kv head's queries; tiles of all kv heads
    int page_shift;
    int bound;               // tokens that a row of the table has room for
    // Workgroup w leaves the part that starts a group in slot 2w + 1 and one
    // that goes on from the workgroup before it in 2w.
    float* parts;            // [slots][tile][dim]
    float2* part_sums;       // [slots][tile]: reference (log2) and sum
    int2* spans;             // [batch][groups]: first workgroup of a group, number of parts
    float* scores;           // [batch * q_heads][bound], log2, where weights are tracked
    float2* sums;            // [batch * q_heads], of groups in one part, where they are
};

__device__ __forceinline__ int length_of(const Attend& a, int b) {
    return min(max(a.lengths[b], 0), a.bound);
}

__device__ __forceinline__ int units_of(int n) { return (n + kUnit - 1) / kUnit; }

// Units that starting a group is worth: its queries, page ids and first keys come
// one after the other, and its waves' parts are joined.  A group's units then lie
// behind as many empty ones, and a share of many short groups has fewer units than
// one of a long group (8 kv heads of 128 columns: 256 sequences of up to 200 tokens
// 48.2 -> 42.1 us, 64 of up to 1000 in 4 bits 22.7 -> 20.8).
constexpr int kOpen = 2;

// How units are dealt to workgroups: `rest` of them get one more than the others.
// Beyond one for each CU, workgroups get two units at least: half as many parts
// to join are worth more than a second workgroup's share of the latency (three
// sequences of 1777 tokens in f32: 15.2 us against 15.8; four of up to 4096 in 4
// bits 14.8 against 15.1).
struct Shares {
    uint32_t workers, open, each, rest;
    // units of all groups, and how many groups have any
    __device__ __forceinline__ Shares(uint32_t units, uint32_t groups, uint32_t most) {
        workers = min(most, units <= kCus ? units : max((uint32_t)kCus, (units + 1) / 2));
        // Not where hardly any share has more than one group, and not where both
        // shares and groups are of few units, which are best cut evenly (64 sequences
        // of up to 200 tokens 16.0 us against 18.8).
        open = 4 * groups >= workers && units >= min(2 * groups, 3 * workers) ? kOpen : 0;
        units += open * groups;
        each = workers ? units / workers : 0;
        rest = units - each * workers;
    }
    __device__ __forceinline__ uint32_t start(uint32_t w) const { return w * each + min(w, rest); }
    __device__ __forceinline__ uint32_t worker_of(uint32_t unit) const {
        const uint32_t longer = rest * (each + 1);
        return unit < longer ? unit / (each + 1) : rest + (unit - longer) / each;
    }
};

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// 0 in the place of a reference for nothing, so that differences stay numbers.
__device__ __forceinline__ float or_zero(float m) { return m == -__builtin_inff() ? 0.f : m; }

// An address that all lanes share, kept apart from what a lane adds to it: loads
// then take it from scalar registers and the lane's 32 bits beside it.
using global_ptr = const __attribute__((address_space(1))) uint8_t*;
__device__ __forceinline__ global_ptr shared_address(const void* p, int64_t off) {
    uint64_t at = (uint64_t)p + off;
    asm("" : "+s"(at));
    return (global_ptr)at;
}

// BYTES bytes of memory in registers, from an address aligned to the largest power of
// two that divides BYTES, or to 16.
template <int BYTES>
struct Raw {
    uint32_t w[BYTES < 4 ? 1 : BYTES / 4];
};
// Three words have no more alignment than one (as an alias of a template the
// attribute would be dropped, and 16 bytes promised).
typedef uint32_t three_words __attribute__((ext_vector_type(3), aligned(4)));
template <int BYTES>
__device__ __forceinline__ Raw<BYTES> load_raw(global_ptr p) {
    Raw<BYTES> r;
    if constexpr (BYTES == 0) {
        r.w[0] = 0;
    } else if constexpr (BYTES == 1) {
        r.w[0] = *p;
    } else if constexpr (BYTES == 2) {
        r.w[0] = *reinterpret_cast<const __attribute__((address_space(1))) uint16_t*>(p);
    } else if constexpr (BYTES == 4) {
        r.w[0] = *reinterpret_cast<const __attribute__((address_space(1))) uint32_t*>(p);
    } else if constexpr (BYTES == 12) {
        const auto x = *reinterpret_cast<const __attribute__((address_space(1))) three_words*>(p);
#pragma unroll
        for (int j = 0; j < 3; j++) r.w[j] = x[j];
    } else {
        constexpr int N = BYTES % 16 == 0 ? 4 : 2;  // words of a load
#pragma unroll
        for (int i = 0; i < BYTES / 4; i += N) {
            const auto x = *reinterpret_cast<const __attribute__((address_space(1))) vec<uint32_t, N>*>(p + 4 * i);
#pragma unroll
            for (int j = 0; j < N; j++) r.w[i + j] = x[j];
        }
    }
    return r;
}

// Which columns a lane holds of a row: dim columns are dealt to 16 lanes as
// one piece of 16 * L0 columns (a power of two) and one of 16 * L1 behind it.
template <int D>
struct Deal {
    static constexpr int P0 = D == 192 ? 128 : D == 96 ? 64 : D;
    static constexpr int L0 = P0 / 16, L1 = (D - P0) / 16;
    // the column that tile t of the second product holds in row n
    static __device__ __forceinline__ int column(int t, int n) {
        return t < L0 ? L0 * n + t : P0 + L1 * n + (t - L0);
    }
};

template <typename T>
using Half8 = vec<T, 8>;

__device__ __forceinline__ vec<float, 4> mma(Half8<__bf16> a, Half8<__bf16> b, vec<float, 4> c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ vec<float, 4> mma(Half8<_Float16> a, Half8<_Float16> b, vec<float, 4> c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// o += a (hi + lo / kRest)
template <typename T>
__device__ __forceinline__ void add_product(vec<float, 4>& o, Half8<T> a, Half8<T> hi, Half8<T> lo) {
    if constexpr (kRest<T> == 1.f) {
        o = mma(a, lo, mma(a, hi, o));
    } else {
        // in this order: the other way round the rests of all tiles are made first,
        // and registers spill
        o += mma(a, lo, vec<float, 4>{}) * (1.f / kRest<T>);
        o = mma(a, hi, o);
    }
}

// The keys of a step as a wave holds them: per tile of 16, lane (key = lane %
// 16, g) has a quarter of its key's columns.  Values: 16 bytes of every 64, so
// that four lanes read 64 neighbouring bytes.  Codes: a quarter of the row.
template <typename T, bool MX, int D>
struct Keys {
    static constexpr int N = MX ? 1 : D * (int)sizeof(T) / 64;      // loads
    static constexpr int BYTES = MX ? D / 8 : 16;                   // of each
    static constexpr int BLOCKS = !MX ? 0 : D == 64 || D == 128 ? 1 : 2;  // scales of a lane
    Raw<BYTES> x[N];
    uint32_t scale[BLOCKS ? BLOCKS : 1];

    // row0: the tile's first row, the same for all lanes
    __device__ __forceinline__ void load(const vramc_kv_cache& c, int64_t row0, int lane) {
        const uint32_t g = lane >> 4, n = lane & 15;
        if constexpr (MX) {
            x[0] = load_raw<BYTES>(shared_address(c.k, row0 * (D / 2)) + (n * (D / 2) + g * BYTES));
            const global_ptr s = shared_address(c.k_scale, row0 * (D / kMxBlock));
            const uint32_t at = n * (D / kMxBlock) + g * (D / 4) / kMxBlock;
            scale[0] = s[at];
            // the last lanes of 96 and 192 columns end in their first block
            if constexpr (BLOCKS == 2)
                scale[1] = s[at + ((g * (D / 4) + D / 4 - 1) / kMxBlock - g * (D / 4) / kMxBlock)];
        } else {
            const global_ptr p = shared_address(c.k, row0 * (D * (int)sizeof(T)));
#pragma unroll
            for (int s = 0; s < N; s++)
                x[s] = load_raw<16>(p + (n * (uint32_t)(D * sizeof(T)) + g * 16) + s * 64);
        }
    }
    // The first column of the lane's chunk s.
    static __device__ __forceinline__ int column(int s, int g) {
        return MX ? g * (D / 4) + 8 * s : sizeof(T) == 4 ? 16 * s + 4 * g : 32 * s + 8 * g;
    }
    // Eight columns as a matrix operand.
    __device__ __forceinline__ Half8<T> operand(int s, int g) const {
        vec<uint32_t, 4> r;
        if constexpr (MX) {
            uint32_t sc = scale[0];
            if constexpr (BLOCKS == 2)
                sc = (g * (D / 4) + 8 * s) / kMxBlock > g * (D / 4) / kMxBlock ? scale[1] : scale[0];
#pragma unroll
            for (int i = 0; i < 4; i++) r[i] = mx_pair_at<T>(x[0].w[s], sc, i);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) r[i] = x[s].w[i];
        }
        return __builtin_bit_cast(Half8<T>, r);
    }
};

// The values of a step: lane (n = lane % 16, g) has columns Deal<D> of key
// (j / 4) * 16 + 4g + j % 4 for each j.
template <typename T, bool MX, int D, int KEYS>
struct Values {
    using C = Deal<D>;
    static constexpr int SIZE = MX ? 1 : 2 * (int)sizeof(T);  // half bytes of a value
    static constexpr int B0 = C::L0 * SIZE / 2, B1 = C::L1 * SIZE / 2;
    Raw<B0> x0[KEYS];
    Raw<B1> x1[KEYS];
    uint32_t scale0[MX ? KEYS : 1], scale1[MX && B1 ? KEYS : 1];

    __device__ __forceinline__ void load(const vramc_kv_cache& c, const int64_t* row0, int lane) {
        const uint32_t n = lane & 15, g = lane >> 4;
        constexpr int ROW = D * SIZE / 2, SCALES = D / kMxBlock;
#pragma unroll
        for (int i = 0; i < KEYS / 4; i++) {
            const global_ptr p = shared_address(c.v, row0[i] * ROW);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x0[4 * i + e] = load_raw<B0>(p + (g * (4 * ROW) + n * B0) + e * ROW);
                if constexpr (B1 > 0) x1[4 * i + e] = load_raw<B1>(p + (g * (4 * ROW) + n * B1) + (e * ROW + 16 * B0));
            }
            if constexpr (MX) {
                const global_ptr s = shared_address(c.v_scale, row0[i] * SCALES);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    scale0[4 * i + e] = *(s + (g * (4 * SCALES) + n * C::L0 / kMxBlock) + e * SCALES);
                    if constexpr (B1 > 0)
                        scale1[4 * i + e] = *(s + (g * (4 * SCALES) + (C::P0 + n * C::L1) / kMxBlock) + e * SCALES);
                }
            }
        }
    }
    // Zeros in the place of key j: what lies there may be anything.
    __device__ __forceinline__ void clear(int j, bool gone) {
#pragma unroll
        for (auto& w : x0[j].w) w = gone ? 0 : w;
#pragma unroll
        for (auto& w : x1[j].w) w = gone ? 0 : w;
        if constexpr (MX) {
            scale0[j] = gone ? 0 : scale0[j];
            if constexpr (B1 > 0) scale1[j] = gone ? 0 : scale1[j];
        }
    }
    // Columns 2p and 2p + 1 of the lane's, of key j, in 16 bits each.
    __device__ __forceinline__ uint32_t pair(int p, int j) const {
        const bool first = p < C::L0 / 2;
        const int i = first ? p : p - C::L0 / 2;
        if constexpr (MX) {
            if constexpr (B1 > 0)
                if (!first) return mx_pair_at<T>(x1[j].w[i / 4], scale1[j], i % 4);
            return mx_pair_at<T>(x0[j].w[i / 4], scale0[j], i % 4);
        } else {
            if constexpr (B1 > 0)
                if (!first) return x1[j].w[i];
            return x0[j].w[i];
        }
    }
    __device__ __forceinline__ float value(int t, int j) const {  // f32
        if constexpr (B1 > 0)
            if (t >= C::L0) return __uint_as_float(x1[j].w[t - C::L0]);
        return __uint_as_float(x0[j].w[t]);
    }
};

// Tiles of query heads that a wave takes at once: two where a kv head has more
// than 16 and the registers hold their queries and sums beside the keys (all but
// two registers of them, for 128 columns of 16 bits), so that up to 32 heads read
// the cache once (16 sequences of up to 16384 tokens, 32 heads of 128 columns: 36
// us against 42; 24 of 64 in f32 54 against 71).  4-bit pages are cheap to read and
// dear to convert with fewer waves at it: one tile (24 heads of 128 columns 35 us
// against 41).
constexpr int pair_of(int size, bool mx, int dim, int group) {
    return group > 16 && !mx && size * dim <= (size == 4 ? 512 : 384) ? 2 : 1;
}

// Waves of a SIMD, and so workgroups of a CU, that the registers are to allow and
// that the work is shared among.  Two cap the registers at 256, which also keeps
// the sums in ordinary ones instead of accumulation registers, from where every
// rescaling would have to copy them; with three, 128 columns spill (16 sequences
// of up to 32768 tokens: 286 us against 276).  Rows of 4 bits are short and need
// the third for the bytes under way (the same sequences: 93 us against 94; of
// 16384 tokens 34 against 38 with 64 columns, 54 against 62 with 96); the widest
// rows fill one wave's registers.
constexpr int waves_of_simd(int size, bool mx, int dim, int pair) {
    if (pair == 2) return size * dim <= 256 ? 2 : 1;
    if (mx) return dim <= 128 ? 3 : 2;
    return dim <= (size == 4 ? 128 : 192) ? 2 : 1;
}

template <typename T, bool MX, int D, int PAIR>
__global__ void __launch_bounds__(kThreads, waves_of_simd(sizeof(T), MX, D, PAIR)) attend_kernel(Attend a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int TILES = F32 ? 1 : 2;       // of 16 keys in a step
    constexpr int STEP = 16 * TILES, KEYS = 4 * TILES;
    constexpr int NT = D / 16;               // tiles of the output
    using C = Deal<D>;
    __shared__ int wave_units[kWaves], wave_some[kWaves], place[2];
    constexpr int JOIN = NT > 12 ? NT / 2 : NT;  // tiles that are joined at once, in 64 KB
    __shared__ float part[kWaves][4][JOIN][64], part_of[kWaves][2][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4;

    // this workgroup's share: each thread counts some sequences' units
    const int each = (a.batch + kThreads - 1) / kThreads, b0 = threadIdx.x * each;
    int mine = 0, some = 0, units_before = 0, some_before = 0, all_units = 0, all_some = 0;
    if (a.batch == 1) {  // nothing to count
        all_units = units_of(length_of(a, 0));
        all_some = all_units > 0;
    } else {
        for (int i = b0; i < min(b0 + each, a.batch); i++) {
            const int units = units_of(length_of(a, i));
            mine += units;
            some += units > 0;
        }
        const int sum = wave_scan(mine), have = wave_scan(some);
        if (lane == 63) {
            wave_units[wave] = sum;
            wave_some[wave] = have;
        }
        __syncthreads();
        units_before = sum - mine;
        some_before = have - some;
#pragma unroll
        for (int w = 0; w < kWaves; w++) {
            units_before += w < wave ? wave_units[w] : 0;
            some_before += w < wave ? wave_some[w] : 0;
            all_units += wave_units[w];
            all_some += wave_some[w];
        }
    }
    const Shares shares(__builtin_amdgcn_readfirstlane(all_units) * (uint32_t)a.groups,
                        __builtin_amdgcn_readfirstlane(all_some) * (uint32_t)a.groups, gridDim.x);
    const int open = shares.open;
    for (int i = blockIdx.x; i < a.batch; i += gridDim.x)  // nothing to attend to
        if (length_of(a, i) == 0) {
            T* to = static_cast<T*>(a.out) + (int64_t)i * a.q_heads * D;
            for (int x = threadIdx.x; x < a.q_heads * D; x += kThreads) to[x] = (T)0.f;
            for (int x = threadIdx.x; x < a.groups; x += kThreads) a.spans[(int64_t)i * a.groups + x] = make_int2(0, 0);
        }
    if (blockIdx.x >= shares.workers) return;
    uint32_t unit = shares.start(blockIdx.x);
    const uint32_t stop = shares.start(blockIdx.x + 1);
    int b = 0, off = (int)unit;
    if (a.batch > 1) {
        const uint32_t before = (uint32_t)(units_before + open * some_before) * a.groups;
        if (unit >= before && unit - before < (uint32_t)(mine + open * some) * a.groups) {
            uint32_t in = unit - before;
            int i = b0;
            for (;; i++) {
                const int units = units_of(length_of(a, i));
                const uint32_t x = units ? (uint32_t)(units + open) * a.groups : 0;
                if (in < x) break;
                in -= x;
            }
            place[0] = i;
            place[1] = (int)in;
        }
        __syncthreads();
        b = __builtin_amdgcn_readfirstlane(place[0]);
        off = __builtin_amdgcn_readfirstlane(place[1]);
    }
    const float scale = a.scale * kLog2e;
    int n = __builtin_amdgcn_readfirstlane(length_of(a, b));

    while (unit < stop) {
        const int units = units_of(n), cost = units + open;
        const int group = off / cost, in = off - group * cost;
        const int dealt = min((uint32_t)(cost - in), stop - unit);
        const int first_unit = max(in - open, 0), here = in + dealt - open - first_unit;
        if (here <= 0) break;  // the share ends in a group's empty units
        const int h = group / a.head_tiles, first_head = group % a.head_tiles * a.tile;
        const int start = first_unit * kUnit, end = min(n, (first_unit + here) * kUnit);
        const bool opens = in <= open, alone = here == units;
        if (opens && threadIdx.x == 0)
            a.spans[(int64_t)b * a.groups + group] =
                make_int2(blockIdx.x, alone ? 1 : shares.worker_of(unit + (cost - in) - 1) - blockIdx.x + 1);
        const auto head_of = [&](int r) { return first_head + 16 * r + (lane & 15); };
        const auto live = [&](int r) { return head_of(r) < a.group; };
        const auto q_row = [&](int r) { return (int64_t)b * a.q_heads + h * a.group + head_of(r); };

        // Page ids of 64 of this wave's tiles of 16 keys, one a lane; the next 64 are
        // fetched while these are used.
        const int steps = (end - start + STEP - 1) / STEP;
        const auto page_ids = [&](int window) {
            const int tile = window * 64 + lane;
            const int key = start + (wave + kWaves * (tile / TILES)) * STEP + tile % TILES * 16;
            int id = -1;
            if (key < end) id = a.table[b * a.table_row + (key >> a.page_shift)];
            return (uint32_t)id < (uint32_t)a.c.pages ? id : -1;
        };
        int window = 0, ids = page_ids(0), next_ids = page_ids(1);

        // the queries, in the keys' order of columns; columns of the tiles beyond the
        // group repeat its first head, and are not written anywhere
        Half8<T> q[PAIR][F32 ? 1 : D / 32];
        vec<float, 4> qf[PAIR][F32 ? D / 16 : 1];
#pragma unroll
        for (int r = 0; r < PAIR; r++) {
            constexpr int N = F32 ? 4 : 8;
            const T* p = static_cast<const T*>(a.q) + b * a.q_seq +
                         (int64_t)(h * a.group + (live(r) ? head_of(r) : first_head)) * a.q_head;
            const auto take = [&](int s, auto& x) {
                const T* from = p + Keys<T, MX, D>::column(s, g);
                if (a.q_wide) {
                    x = *reinterpret_cast<const vec<T, N>*>(from);
                } else {
#pragma unroll
                    for (int i = 0; i < N; i++) x[i] = from[i];
                }
            };
#pragma unroll
            for (int s = 0; s < D / (F32 ? 16 : 32); s++) {
                if constexpr (F32) take(s, qf[r][s]);
                else take(s, q[r][s]);
            }
        }

        // The step at hand.  As soon as its keys are multiplied the next step's take
        // their registers, and so with the values, so that some of both is always
        // under way.
        Keys<T, MX, D> k[TILES];
        Values<T, MX, D, KEYS> v;
        int page[TILES];
        int64_t row[TILES];
        const auto find = [&](int t) {  // page 0 stands in for a missing one
            const int tile = t / kWaves * TILES;
            if (tile / 64 != window) {
                ids = next_ids;
                next_ids = page_ids(++window + 1);
            }
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                page[i] = __builtin_amdgcn_readlane(ids, tile % 64 + i);
                row[i] = (((int64_t)max(page[i], 0) * a.c.kv_heads + h) << a.page_shift) +
                           ((start + t * STEP + i * 16) & (a.c.page_size - 1));
            }
        };
        const auto load_keys = [&] {
#pragma unroll
            for (int i = 0; i < TILES; i++) k[i].load(a.c, row[i], lane);
        };

        vec<float, 4> o[PAIR][NT] = {};
        float m[PAIR], from[PAIR] = {}, l[PAIR] = {};
#pragma unroll
        for (int r = 0; r < PAIR; r++) m[r] = -__builtin_inff();
        if (wave < steps) {
            find(wave);
            load_keys();
            v.load(a.c, row, lane);
        }
        for (int t = wave; t < steps; t += kWaves) {
            const int key0 = start + t * STEP;
            bool whole = key0 + STEP <= end;
            bool there[TILES];
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                there[i] = page[i] >= 0;
                whole &= there[i];
            }
            vec<float, 4> s[PAIR][TILES] = {};
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                if constexpr (F32) {
                    // Four sums of a quarter of the columns each, then those: one sum of
                    // all is two to three times as far off (three sequences of up to
                    // 1777 tokens, 96 columns: 1.1e-6 against 4.5e-7 of the output's
                    // norm; elementary f32 operations 5.3e-7), and no faster.
                    vec<float, 4> quarter[PAIR][4] = {};
#pragma unroll
                    for (int c = 0; c < D / 16; c++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
#pragma unroll
                            for (int r = 0; r < PAIR; r++)
                                quarter[r][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                    __uint_as_float(k[i].x[c].w[e]), qf[r][c][e], quarter[r][e], 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < PAIR; r++)
                        s[r][i] = (quarter[r][0] + quarter[r][1]) + (quarter[r][2] + quarter[r][3]);
                } else {
#pragma unroll
                    for (int c = 0; c < D / 32; c++) {
                        const auto x = k[i].operand(c, g);
#pragma unroll
                        for (int r = 0; r < PAIR; r++) s[r][i] = mma(x, q[r][c], s[r][i]);
                    }
                }
            }
            const bool more = t + kWaves < steps;
            if (more) {
                find(t + kWaves);
                load_keys();
            }
            if (!whole) {
#pragma unroll
                for (int j = 0; j < KEYS; j++) v.clear(j, !there[j >> 2] || key0 + 16 * (j >> 2) + 4 * g + (j & 3) >= end);
            }
            float p[PAIR][KEYS];
#pragma unroll
            for (int r = 0; r < PAIR; r++) {
#pragma unroll
                for (int i = 0; i < TILES; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[r][i][e] *= scale;
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < TILES; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (!there[i] || key0 + 16 * i + 4 * g + e >= end) s[r][i][e] = -__builtin_inff();
                }
                if (a.scores && live(r)) {
#pragma unroll
                    for (int i = 0; i < TILES; i++)
                        if (key0 + 16 * i < a.bound)
                            *reinterpret_cast<vec<float, 4>*>(a.scores + q_row(r) * a.bound + key0 + 16 * i + 4 * g) = s[r][i];
                }
                float top = -__builtin_inff();
#pragma unroll
                for (int i = 0; i < TILES; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) top = fmaxf(top, s[r][i][e]);
                if (__builtin_expect(__any(top > m[r] + kSlack<T>), 0)) {
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    if (top > m[r] + kSlack<T>) {
                        from[r] = or_zero(top - kBelow<T>);
                        const float keep = exp2_of(m[r] - from[r]);
                        l[r] *= keep;
#pragma unroll
                        for (int i = 0; i < NT; i++) o[r][i] *= keep;
                        m[r] = top - kBelow<T>;
                    }
                }
#pragma unroll
                for (int j = 0; j < KEYS; j++) {
                    p[r][j] = exp2_of(s[r][j >> 2][j & 3] - from[r]);
                    l[r] += p[r][j];
                }
            }
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < KEYS; j++)
#pragma unroll
                    for (int i = 0; i < NT; i++)
#pragma unroll
                        for (int r = 0; r < PAIR; r++)
                            o[r][i] = __builtin_amdgcn_mfma_f32_16x16x4f32(v.value(i, j), p[r][j], o[r][i], 0, 0, 0);
            } else {
                Half8<T> hi[PAIR], lo[PAIR];
#pragma unroll
                for (int r = 0; r < PAIR; r++) {
                    vec<T, 2> hi2[4], lo2[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const vec<float, 2> w = {p[r][2 * j], p[r][2 * j + 1]};
                        hi2[j] = __builtin_convertvector(w, vec<T, 2>);
                        lo2[j] = __builtin_convertvector((w - __builtin_convertvector(hi2[j], vec<float, 2>)) * kRest<T>, vec<T, 2>);
                    }
                    hi[r] = __builtin_bit_cast(Half8<T>, hi2);
                    lo[r] = __builtin_bit_cast(Half8<T>, lo2);
                }
#pragma unroll
                for (int i = 0; i < NT / 2; i++) {
                    vec<uint32_t, 4> even, odd;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const uint32_t y = v.pair(i, 2 * j), z = v.pair(i, 2 * j + 1);
                        even[j] = __builtin_amdgcn_perm(z, y, 0x05040100);
                        odd[j] = __builtin_amdgcn_perm(z, y, 0x07060302);
                    }
                    const auto e = __builtin_bit_cast(Half8<T>, even), f = __builtin_bit_cast(Half8<T>, odd);
#pragma unroll
                    for (int r = 0; r < PAIR; r++) {
                        add_product(o[r][2 * i], e, hi[r], lo[r]);
                        add_product(o[r][2 * i + 1], f, hi[r], lo[r]);
                    }
                }
            }
            if (more) v.load(a.c, row, lane);
        }
#pragma unroll
        for (int r = 0; r < PAIR; r++) {
            l[r] += __shfl_xor(l[r], 16);
            l[r] += __shfl_xor(l[r], 32);
        }

        // The waves' parts, joined through LDS: wave w takes register w of every tile,
        // neighbouring columns of a lane, and writes them.  (In two rounds of halves,
        // one wave writing all: 256 sequences of up to 200 tokens in 4 bits 30 us
        // against 26, 16 of up to 32768 276 against 274.)
#pragma unroll
        for (int r = 0; r < PAIR; r++) {
            float top = -__builtin_inff(), sum = 0.f, w[kWaves], x[NT] = {};
#pragma unroll
            for (int c = 0; c < NT; c += JOIN) {
                __syncthreads();  // what was there has been read
#pragma unroll
                for (int e = 0; e < 4; e++)
#pragma unroll
                    for (int i = 0; i < JOIN; i++) part[wave][e][i][lane] = o[r][c + i][e];
                if (c == 0) {
                    part_of[wave][0][lane] = m[r];
                    part_of[wave][1][lane] = l[r];
                }
                __syncthreads();
                if (c == 0) {
#pragma unroll
                    for (int u = 0; u < kWaves; u++) top = fmaxf(top, w[u] = part_of[u][0][lane]);
#pragma unroll
                    for (int u = 0; u < kWaves; u++) {
                        w[u] = exp2_of(w[u] - or_zero(top));
                        sum += part_of[u][1][lane] * w[u];
                    }
                }
#pragma unroll
                for (int i = 0; i < JOIN; i++)
#pragma unroll
                    for (int u = 0; u < kWaves; u++) x[c + i] += part[u][wave][i][lane] * w[u];
            }
            if (!live(r)) continue;
            const int column = 4 * g + wave;
            if (alone) {
                if (a.scores && wave == 0 && g == 0) a.sums[q_row(r)] = make_float2(top, sum);
                const float unit_sum = sum == 0.f ? 0.f : 1.f / sum;
                T* to = static_cast<T*>(a.out) + q_row(r) * D;
#pragma unroll
                for (int i = 0; i < NT; i++) to[C::column(i, column)] = (T)(sum == 0.f ? 0.f : x[i] * unit_sum);
            } else {
                const int64_t at = (int64_t)(2 * blockIdx.x + opens) * a.tile + 16 * r + (lane & 15);
                if (wave == 0 && g == 0) a.part_sums[at] = make_float2(top, sum);
                float* to = a.parts + at * D;
#pragma unroll
                for (int i = 0; i < NT; i++) to[C::column(i, column)] = x[i];
            }
        }
        unit += dealt;
        off += dealt;
        if (off == cost * a.groups) {  // on to the next sequence that has tokens
            off = 0;
            while (unit < stop && (n = __builtin_amdgcn_readfirstlane(length_of(a, ++b))) == 0) {}
        }
    }
}

// What is left when all parts are there.  The first blocks join the parts; the
// others add the weights of 1024 tokens of a kv head to their mass, from the
// scores that the first launch left.  Where the workgroups make some eight parts
// of a group or fewer, a thread joins four columns of a query head; where more, a
// block joins 32 columns, 32 parts at a time: one sequence of 131072 tokens takes
// 30 us in place of 80, three of 1777 in f32 15.1 in place of 17.1, but 64 of 2049
// (two parts of each of 768 heads) 33.7 us in place of 28.7.
constexpr int kFewParts = 8;
constexpr int kJoinColumns = 32, kJoinLanes = kJoinColumns / 4, kJoinParts = kThreads / kJoinLanes;
constexpr int kMassKeys = 4 * kThreads, kMassHeads = kThreads / 16;

// The rows of a query head's parts, in order: slot 2w + 1 of the workgroup that
// opens it, then slots 2w.
struct Parts {
    int64_t first;
    int count, tile;
    __device__ __forceinline__ Parts(const Attend& a, int b, int q_head) {
        const int h = q_head / a.group, in = q_head - h * a.group;
        const int2 span = a.spans[(int64_t)b * a.groups + h * a.head_tiles + in / a.tile];
        tile = a.tile;
        first = (int64_t)2 * span.x * tile + in % tile;
        count = span.y;
    }
    __device__ __forceinline__ int64_t row(int i) const { return first + (i ? 2 * i : 1) * tile; }
};

// The largest reference and the sum over a query head's parts, by LANES lanes.
template <int LANES>
__device__ __forceinline__ float2 total_of(const float2* sums, const Parts& parts, int lane) {
    float m = -__builtin_inff(), l = 0.f;
    for (int i = lane; i < parts.count; i += LANES) {
        const float2 x = sums[parts.row(i)];
        const float top = fmaxf(m, x.x);
        l = l * exp2_of(m - or_zero(top)) + x.y * exp2_of(x.x - or_zero(top));
        m = top;
    }
    float top = m;
#pragma unroll
    for (int x = LANES / 2; x; x /= 2) top = fmaxf(top, __shfl_xor(top, x));
    l *= exp2_of(m - or_zero(top));
#pragma unroll
    for (int x = LANES / 2; x; x /= 2) l += __shfl_xor(l, x);
    return make_float2(or_zero(top), l);
}

template <typename T>
__device__ __forceinline__ void join_few(const Attend& a, int block) {
    const int dim = a.c.head_dim;
    const int64_t at = 4 * ((int64_t)block * kThreads + threadIdx.x), q_row = at / dim;
    if (q_row >= (int64_t)a.batch * a.q_heads) return;
    const Parts parts(a, (int)(q_row / a.q_heads), (int)(q_row % a.q_heads));
    if (parts.count <= 1) return;
    const float* in = a.parts + (at - q_row * dim);
    vec<float, 4> x = {};
    float m = -__builtin_inff(), l = 0.f;
    for (int i = 0; i < parts.count; i += 4) {
        vec<float, 4> y[4];
        float2 ml[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int64_t row = parts.row(min(i + u, parts.count - 1));
            y[u] = *reinterpret_cast<const vec<float, 4>*>(in + row * dim);
            ml[u] = a.part_sums[row];
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (i + u < parts.count) {
                const float top = fmaxf(m, ml[u].x);
                const float keep = exp2_of(m - or_zero(top)), w = exp2_of(ml[u].x - or_zero(top));
                x = x * keep + y[u] * w;
                l = l * keep + ml[u].y * w;
                m = top;
            }
    }
    T* to = static_cast<T*>(a.out) + at;
#pragma unroll
    for (int e = 0; e < 4; e++) to[e] = (T)(l == 0.f ? 0.f : x[e] / l);
}

template <typename T>
__device__ __forceinline__ void join(const Attend& a, int block) {
    __shared__ float sum[kWaves][kJoinColumns];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, dim = a.c.head_dim;
    const int q_row = block / (dim / kJoinColumns), first = block % (dim / kJoinColumns) * kJoinColumns;
    const Parts parts(a, q_row / a.q_heads, q_row % a.q_heads);
    if (parts.count <= 1) return;
    const float* in = a.parts + first + threadIdx.x % kJoinLanes * 4;
    // eight lanes take a part's columns, 32 parts at a time, four of them under way
    vec<float, 4> x = {};
    const float2 all = total_of<64>(a.part_sums, parts, lane);
    for (int i = threadIdx.x / kJoinLanes; i < parts.count; i += 4 * kJoinParts) {
        vec<float, 4> y[4];
        float w[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int64_t row = parts.row(min(i + u * kJoinParts, parts.count - 1));
            y[u] = *reinterpret_cast<const vec<float, 4>*>(in + row * dim);
            w[u] = a.part_sums[row].x;
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (i + u * kJoinParts < parts.count) x += exp2_of(w[u] - all.x) * y[u];
    }
#pragma unroll
    for (int d = kJoinLanes; d < 64; d *= 2)
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] += __shfl_xor(x[e], d);
    if (lane < kJoinLanes)
#pragma unroll
        for (int e = 0; e < 4; e++) sum[wave][lane * 4 + e] = x[e];
    __syncthreads();
    if (threadIdx.x < kJoinColumns) {
        float o = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; w++) o += sum[w][threadIdx.x];
        static_cast<T*>(a.out)[(int64_t)q_row * dim + first + threadIdx.x] = (T)(all.y == 0.f ? 0.f : o / all.y);
    }
}

__device__ __forceinline__ void add_mass(const Attend& a, int block) {
    __shared__ float2 total[kMassHeads];
    const int tiles = (a.bound + kMassKeys - 1) / kMassKeys;
    const int tile = block % tiles, b = block / tiles / a.c.kv_heads, h = block / tiles % a.c.kv_heads;
    const int n = length_of(a, b);
    if (tile * kMassKeys >= n) return;
    const int64_t first = (int64_t)b * a.q_heads + h * a.group;
    const int key = tile * kMassKeys + 4 * threadIdx.x, at = min(key, a.bound - 4);
    const int page = a.table[b * a.table_row + (at >> a.page_shift)];
    vec<float, 4> w = {};
    for (int base = 0; base < a.group; base += kMassHeads) {
        const int heads = min(a.group - base, kMassHeads);
        vec<float, 4> s[kMassHeads];
#pragma unroll
        for (int i = 0; i < kMassHeads; i++)
            if (i < heads) s[i] = *reinterpret_cast<const vec<float, 4>*>(a.scores + (first + base + i) * a.bound + at);
        if (base) __syncthreads();
        // the totals of 16 heads at once, 16 lanes each
        const int i = threadIdx.x / 16;
        if (i < heads) {
            const Parts parts(a, b, h * a.group + base + i);
            const float2 t = parts.count > 1 ? total_of<16>(a.part_sums, parts, threadIdx.x % 16)
                                             : a.sums[first + base + i];
            if (threadIdx.x % 16 == 0) total[i] = make_float2(or_zero(t.x), t.y == 0.f ? 0.f : 1.f / t.y);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kMassHeads; i++)
            if (i < heads && total[i].y != 0.f)
#pragma unroll
                for (int e = 0; e < 4; e++) w[e] += exp2_of(s[i][e] - total[i].x) * total[i].y;
    }
    // By neighbouring lanes to neighbouring tokens: as each lane's four, the additions
    // of 16 sequences of up to 32768 tokens, 40 heads, took 25 us longer (393 against
    // 368 us in all).
    __shared__ __attribute__((aligned(16))) float sum[kMassKeys];
    __shared__ int64_t places[kThreads];
    const bool there = key < n && page >= 0 && page < a.c.pages;
    *reinterpret_cast<vec<float, 4>*>(sum + 4 * threadIdx.x) = w;
    places[threadIdx.x] =
        there ? (((int64_t)page * a.c.kv_heads + h) << a.page_shift) + (key & (a.c.page_size - 1)) : -1;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int i = e * kThreads + threadIdx.x;
        const int64_t to = places[i / 4];
        if (to >= 0 && tile * kMassKeys + i < n) unsafeAtomicAdd(a.c.mass + to + i % 4, sum[i]);
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) finish_kernel(Attend a, int joins, bool few) {
    if ((int)blockIdx.x >= joins) add_mass(a, blockIdx.x - joins);
    else if (few) join_few<T>(a, blockIdx.x);
    else join<T>(a, blockIdx.x);
}

template <typename T, bool MX, int D>
int launch(const Attend& a, int workers, hipStream_t stream) {
    const dim3 grid((unsigned)workers), block(kThreads);
    if constexpr (pair_of(sizeof(T), MX, D, 17) == 2) {
        if (a.tile == 32) hipLaunchKernelGGL((attend_kernel<T, MX, D, 2>), grid, block, 0, stream, a);
    }
    if (a.tile == 16) hipLaunchKernelGGL((attend_kernel<T, MX, D, 1>), grid, block, 0, stream, a);
    if (const int rc = (int)hipGetLastError()) return rc;
    const bool few = workers <= (int64_t)a.batch * a.groups * kFewParts;
    const int64_t rows = (int64_t)a.batch * a.q_heads;
    const int64_t joins = a.bound <= kUnit ? 0
                          : few                        ? (rows * (D / 4) + kThreads - 1) / kThreads
                                                       : rows * (D / kJoinColumns);
    const int64_t tiles = a.scores ? (int64_t)((a.bound + kMassKeys - 1) / kMassKeys) * a.batch * a.c.kv_heads : 0;
    if (joins + tiles == 0) return 0;
    hipLaunchKernelGGL((finish_kernel<T>), dim3((unsigned)(joins + tiles)), dim3(kThreads), 0, stream, a,
                       (int)joins, few);
    return (int)hipGetLastError();
}

template <typename T, bool MX>
int attend(const Attend& a, int workers, hipStream_t stream) {
    switch (a.c.head_dim) {
        case 64: return launch<T, MX, 64>(a, workers, stream);
        case 96: return launch<T, MX, 96>(a, workers, stream);
        case 128: return launch<T, MX, 128>(a, workers, stream);
        case 192: return launch<T, MX, 192>(a, workers, stream);
        default: return launch<T, MX, 256>(a, workers, stream);
    }
}

// Query rows and units of a call: a grid of both launches' blocks for either
// stays below 2^32 threads, and shares and row lengths are counted in 32 bits.
constexpr int64_t kMaxRows = 1 << 22, kMaxUnits = 1 << 26;

// What a call needs of memory besides its arguments, and its workgroups: as many
// as the CUs hold, but not more than there can be units.
struct Plan {
    int64_t groups, units;  // of a sequence; of all, at most
    int workers, tile;
    int64_t parts, part_sums, spans, scores, sums;  // bytes
    int64_t bytes() const { return parts + part_sums + spans + scores + sums; }
};
Plan plan(const vramc_kv_cache& c, int q_heads, int table_width, int batch, bool track) {
    Plan p;
    const int64_t bound = (int64_t)table_width * c.page_size, rows = (int64_t)batch * q_heads;
    const int size = c.dtype == RANS_X_F32 ? 4 : 2, group = q_heads / c.kv_heads;
    const int pair = pair_of(size, c.mx, c.head_dim, group);
    p.tile = 16 * pair;
    p.groups = (int64_t)c.kv_heads * ((group + p.tile - 1) / p.tile);
    p.units = (bound + kUnit - 1) / kUnit * p.groups * batch;
    const int resident = kCus * waves_of_simd(size, c.mx, c.head_dim, pair);
    p.workers = (int)(p.units < resident ? (p.units ? p.units : 1) : resident);
    p.parts = (int64_t)p.workers * 2 * p.tile * c.head_dim * 4;
    p.part_sums = (int64_t)p.workers * 2 * p.tile * 8;
    p.spans = (p.groups * batch * 8 + 15) / 16 * 16;
    p.scores = track ? rows * bound * 4 : 0;
    p.sums = track ? rows * 8 : 0;
    return p;
}

}  // namespace

extern "C" int64_t vramc_kv_attend_workspace(const vramc_kv_cache* c, int q_heads, int table_width,
                                             int batch, int track) {
    if (const int rc = check_cache(c)) return rc;
    if (q_heads <= 0 || q_heads % c->kv_heads || table_width < 0 || batch < 0) return RANS_EARG;
    if ((int64_t)table_width * c->page_size > kMaxTokens || (int64_t)batch * q_heads > kMaxRows)
        return RANS_EARG;
    const Plan p = plan(*c, q_heads, table_width, batch, track);
    if (p.units > kMaxUnits) return RANS_EARG;
    return p.bytes();
}

extern "C" int vramc_kv_attend(const vramc_kv_cache* c, const void* q, int64_t q_seq,
                               int64_t q_head, int q_heads, const int32_t* table,
                               int64_t table_row, int table_width, const int32_t* lengths,
                               int batch, float scale, int track, void* out, void* workspace,
                               int64_t workspace_bytes, hipStream_t stream) {
    const int64_t need = vramc_kv_attend_workspace(c, q_heads, table_width, batch, track);
    if (need < 0) return (int)need;
    if (batch == 0) return 0;
    if (!q || !out || !lengths || (table_width && !table) || (track && !c->mass)) return RANS_EARG;
    if (!workspace || workspace_bytes < need) return RANS_EWORKSPACE;
    if ((uintptr_t)workspace % 16) return RANS_EARG;
    const Plan p = plan(*c, q_heads, table_width, batch, track);
    auto* work = static_cast<uint8_t*>(workspace);
    const auto take = [&](int64_t bytes) {
        auto* at = work;
        work += bytes;
        return static_cast<void*>(at);
    };
    const int64_t size = c->dtype == RANS_X_F32 ? 4 : 2;
    const bool wide = ((uintptr_t)q | (uintptr_t)(q_seq * size) | (uintptr_t)(q_head * size)) % 16 == 0;
    Attend a{*c, q, q_seq, q_head, wide, q_heads, q_heads / c->kv_heads, table, table_row, lengths, batch,
             scale, out, p.tile, (int)(p.groups / c->kv_heads), (int)p.groups,
             __builtin_ctz(c->page_size), table_width * c->page_size, nullptr, nullptr, nullptr, nullptr, nullptr};
    a.parts = static_cast<float*>(take(p.parts));
    a.part_sums = static_cast<float2*>(take(p.part_sums));
    a.spans = static_cast<int2*>(take(p.spans));
    if (p.scores) {
        a.scores = static_cast<float*>(take(p.scores));
        a.sums = static_cast<float2*>(take(p.sums));
    }
    if (c->dtype == RANS_X_F32) return attend<float, false>(a, p.workers, stream);
    if (c->dtype == RANS_X_BF16)
        return c->mx ? attend<__bf16, true>(a, p.workers, stream) : attend<__bf16, false>(a, p.workers, stream);
    return c->mx ? attend<_Float16, true>(a, p.workers, stream) : attend<_Float16, false>(a, p.workers, stream);
}
