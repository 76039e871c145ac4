// Attention of one new token of each sequence over a paged cache.
//
// What bounds it is reading the keys and values once; a token's 4*dim*group
// operations are few.  Everything else is arranged so that a wave only loads
// and multiplies:
//
//  - The query heads of a kv head are the 16 columns of the matrix cores'
//    tiles, so keys and values are read once for up to 16 of them.  Scores are
//    made transposed, S^T = K Q^T (16 keys x 16 heads): a lane then holds, for
//    one head, the scores of keys 4g..4g+3 of each tile (g = lane / 16), and
//    that is just how the second product O^T = V^T P^T wants its right operand
//    if its inner index runs over the keys in the order (tile, g, 0..3).  So
//    weights never leave the lane that made them, softmax needs a lane's own
//    values and two exchanges for the maximum, and no LDS is touched.
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
//
// The length is split over workgroups, whose waves take turns of 32 keys (16
// in f32); parts are joined in a second launch, which also adds the weights to
// the tokens' mass where that is tracked.
#include "kv_device.h"

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kHeadTile = 16;     // query heads of a workgroup
constexpr int kMaxChunk = 4096;   // keys of a workgroup: its waves keep their page ids in lanes
constexpr float kLog2e = 1.4426950408889634f;

// The reference is set this far below the largest score so far, and again when
// a score exceeds it by Slack (both log2).  f16 weights begin at 2^13, so that
// they keep their bits down to 2^-27 of the largest: its smallest step is
// 2^-24, and the largest value 2^16.
template <typename T>
constexpr float kBelow = std::is_same_v<T, _Float16> ? 13.f : 0.f;
template <typename T>
constexpr float kSlack = std::is_same_v<T, _Float16> ? 15.f : 8.f;

struct Attend {
    vramc_kv_cache c;
    const void* q;
    int64_t q_seq, q_head;
    int q_heads, group;
    const int32_t* table;
    int64_t table_row;
    int table_width;
    const int32_t* lengths;
    int batch;
    float scale;
    void* out;
    int chunk, splits;       // keys of a part, parts of the longest possible sequence
    int head_tiles;
    int page_shift;
    int bound;               // tokens that a row of the table has room for
    float* scores;           // [batch * q_heads][bound], log2, where weights are tracked
    float* parts;            // [batch * q_heads][splits][dim]
    float2* sums;            // [batch * q_heads][splits]: reference (log2) and sum
};

__device__ __forceinline__ int length_of(const Attend& a, int b) {
    return min(max(a.lengths[b], 0), a.bound);
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// 0 in the place of a reference for nothing, so that differences stay numbers.
__device__ __forceinline__ float or_zero(float m) { return m == -__builtin_inff() ? 0.f : m; }

// BYTES bytes of memory in registers, from an address aligned to ALIGN.
template <int BYTES>
struct Raw {
    uint32_t w[BYTES < 4 ? 1 : BYTES / 4];
};
template <int BYTES, int ALIGN>
__device__ __forceinline__ Raw<BYTES> load_raw(const uint8_t* p) {
    Raw<BYTES> r;
    if constexpr (BYTES == 0) {
        r.w[0] = 0;
    } else if constexpr (BYTES == 1) {
        r.w[0] = *p;
    } else if constexpr (BYTES == 2) {
        r.w[0] = *reinterpret_cast<const uint16_t*>(p);
    } else {
        __builtin_memcpy(r.w, __builtin_assume_aligned(p, ALIGN), BYTES);
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
            const uint8_t* p = static_cast<const uint8_t*>(c.k) + row0 * (D / 2);
            x[0] = load_raw<BYTES, BYTES % 16 == 0 ? 16 : BYTES % 8 == 0 ? 8 : 4>(p + (n * (D / 2) + g * BYTES));
            const uint8_t* s = c.k_scale + row0 * (D / kMxBlock);
            const uint32_t at = n * (D / kMxBlock) + g * (D / 4) / kMxBlock;
            scale[0] = s[at];
            // the last lanes of 96 and 192 columns end in their first block
            if constexpr (BLOCKS == 2)
                scale[1] = s[at + ((g * (D / 4) + D / 4 - 1) / kMxBlock - g * (D / 4) / kMxBlock)];
        } else {
            const uint8_t* p = static_cast<const uint8_t*>(c.k) + row0 * (D * (int)sizeof(T));
#pragma unroll
            for (int s = 0; s < N; s++)
                x[s] = load_raw<16, 16>(p + (n * (uint32_t)(D * sizeof(T)) + g * 16) + s * 64);
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
        constexpr int A0 = B0 < 16 ? B0 : 16, A1 = B1 ? B1 : 1;
#pragma unroll
        for (int j = 0; j < KEYS; j++) {
            const uint8_t* p = static_cast<const uint8_t*>(c.v) + row0[j >> 2] * ROW;
            x0[j] = load_raw<B0, A0>(p + (g * (4 * ROW) + n * B0) + (j & 3) * ROW);
            if constexpr (B1 > 0) x1[j] = load_raw<B1, A1>(p + (g * (4 * ROW) + n * B1) + ((j & 3) * ROW + 16 * B0));
            if constexpr (MX) {
                const uint8_t* s = c.v_scale + row0[j >> 2] * SCALES;
                scale0[j] = *(s + (g * (4 * SCALES) + n * C::L0 / kMxBlock) + (j & 3) * SCALES);
                if constexpr (B1 > 0)
                    scale1[j] = *(s + (g * (4 * SCALES) + (C::P0 + n * C::L1) / kMxBlock) + (j & 3) * SCALES);
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

// Waves of a SIMD that the registers are to allow.  Two cap them at 256, which
// also keeps the sums in ordinary registers instead of accumulation registers,
// from where every rescaling would have to copy them.
template <typename T, int D>
constexpr int kWavesOfSimd = D <= (sizeof(T) == 4 ? 128 : 192) ? 2 : 1;

template <typename T, bool MX, int D>
__global__ void __launch_bounds__(kThreads, (kWavesOfSimd<T, D>)) attend_kernel(Attend a) {
    constexpr bool F32 = sizeof(T) == 4;
    constexpr int TILES = F32 ? 1 : 2;       // of 16 keys in a step
    constexpr int STEP = 16 * TILES, KEYS = 4 * TILES;
    constexpr int NT = D / 16;               // tiles of the output
    constexpr int AHEAD = !MX ? 1 : D == 96 ? 3 : D <= 128 ? 4 : 2;
    using C = Deal<D>;
    const int split = blockIdx.x % a.splits;
    int rest = blockIdx.x / a.splits;
    const int first_head = rest % a.head_tiles * kHeadTile;
    rest /= a.head_tiles;
    const int h = rest % a.c.kv_heads, b = rest / a.c.kv_heads;
    const int n = length_of(a, b), start = split * a.chunk;
    if (start >= n && split) return;
    const int end = min(n, start + a.chunk);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, head = first_head + (lane & 15);
    const bool live = head < a.group;
    const int64_t q_row = (int64_t)b * a.q_heads + h * a.group + head;

    // the queries, in the keys' order of columns; heads beyond the group are zero
    Half8<T> q[F32 ? 1 : D / 32];
    vec<float, 4> qf[F32 ? D / 16 : 1];
    {
        const T* p = static_cast<const T*>(a.q) + b * a.q_seq + (int64_t)(h * a.group + head) * a.q_head;
        if constexpr (F32) {
#pragma unroll
            for (int s = 0; s < D / 16; s++)
#pragma unroll
                for (int i = 0; i < 4; i++) qf[s][i] = live ? p[Keys<T, MX, D>::column(s, g) + i] : 0.f;
        } else {
#pragma unroll
            for (int s = 0; s < D / 32; s++)
#pragma unroll
                for (int i = 0; i < 8; i++) q[s][i] = live ? p[Keys<T, MX, D>::column(s, g) + i] : (T)0.f;
        }
    }

    // page ids of this wave's steps, one tile of 16 keys a lane
    const int steps = end > start ? (end - start + STEP - 1) / STEP : 0;
    int pages = -1;
    {
        const int key = start + (wave + kWaves * (lane / TILES)) * STEP + lane % TILES * 16;
        if (key < end) pages = a.table[b * a.table_row + (key >> a.page_shift)];
        if ((uint32_t)pages >= (uint32_t)a.c.pages) pages = -1;
    }
    // A step's keys and values as they arrive: AHEAD steps are in flight, so that
    // a wave has some 8 KB on the way whatever the type.
    struct Step {
        Keys<T, MX, D> k[TILES];
        Values<T, MX, D, KEYS> v;
        int page[TILES];
        int64_t row[TILES];
    } step[AHEAD];
    const auto find = [&](Step& x, int t) {  // page 0 stands in for a missing one
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            x.page[i] = __builtin_amdgcn_readlane(pages, t / kWaves * TILES + i);
            x.row[i] = (((int64_t)max(x.page[i], 0) * a.c.kv_heads + h) << a.page_shift) +
                       ((start + t * STEP + i * 16) & (a.c.page_size - 1));
        }
    };
    const auto load_keys = [&](Step& x) {
#pragma unroll
        for (int i = 0; i < TILES; i++) x.k[i].load(a.c, x.row[i], lane);
    };

    vec<float, 4> o[NT] = {};
    float m = -__builtin_inff(), from = 0.f, l = 0.f;
    const float scale = a.scale * kLog2e;
#pragma unroll
    for (int u = 0; u < AHEAD; u++)
        if (wave + u * kWaves < steps) {
            find(step[u], wave + u * kWaves);
            load_keys(step[u]);
            step[u].v.load(a.c, step[u].row, lane);
        }
    const auto compute = [&](Step& x, int t) {
        const int key0 = start + t * STEP;
        bool whole = key0 + STEP <= end;
        bool there[TILES];
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            there[i] = x.page[i] >= 0;
            whole &= there[i];
        }
        vec<float, 4> s[TILES] = {};
#pragma unroll
        for (int i = 0; i < TILES; i++) {
            if constexpr (F32) {
#pragma unroll
                for (int c = 0; c < D / 16; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        s[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(x.k[i].x[c].w[e]),
                                                                    qf[c][e], s[i], 0, 0, 0);
            } else {
#pragma unroll
                for (int c = 0; c < D / 32; c++) s[i] = mma(x.k[i].operand(c, g), q[c], s[i]);
            }
        }
        const int next = t + AHEAD * kWaves;
        if (next < steps) {
            find(x, next);
            load_keys(x);
        }
#pragma unroll
        for (int i = 0; i < TILES; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[i][e] *= scale;
        if (!whole) {
#pragma unroll
            for (int i = 0; i < TILES; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const bool gone = !there[i] || key0 + 16 * i + 4 * g + e >= end;
                    if (gone) s[i][e] = -__builtin_inff();
                    x.v.clear(4 * i + e, gone);
                }
        }
        if (a.scores && live) {
#pragma unroll
            for (int i = 0; i < TILES; i++)
                if (key0 + 16 * i < a.bound)
                    *reinterpret_cast<vec<float, 4>*>(a.scores + q_row * a.bound + key0 + 16 * i + 4 * g) = s[i];
        }
        float top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < TILES; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) top = fmaxf(top, s[i][e]);
        if (__builtin_expect(__any(top > m + kSlack<T>), 0)) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            if (top > m + kSlack<T>) {
                from = or_zero(top - kBelow<T>);
                const float keep = exp2_of(m - from);
                l *= keep;
#pragma unroll
                for (int i = 0; i < NT; i++) o[i] *= keep;
                m = top - kBelow<T>;
            }
        }
        float p[KEYS];
#pragma unroll
        for (int j = 0; j < KEYS; j++) {
            p[j] = exp2_of(s[j >> 2][j & 3] - from);
            l += p[j];
        }
        if constexpr (F32) {
#pragma unroll
            for (int j = 0; j < KEYS; j++)
#pragma unroll
                for (int i = 0; i < NT; i++)
                    o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v.value(i, j), p[j], o[i], 0, 0, 0);
        } else {
            vec<T, 2> hi2[4], lo2[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const vec<float, 2> w = {p[2 * j], p[2 * j + 1]};
                hi2[j] = __builtin_convertvector(w, vec<T, 2>);
                lo2[j] = __builtin_convertvector(w - __builtin_convertvector(hi2[j], vec<float, 2>), vec<T, 2>);
            }
            const auto hi = __builtin_bit_cast(Half8<T>, hi2), lo = __builtin_bit_cast(Half8<T>, lo2);
#pragma unroll
            for (int i = 0; i < NT / 2; i++) {
                vec<uint32_t, 4> even, odd;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t y = x.v.pair(i, 2 * j), z = x.v.pair(i, 2 * j + 1);
                    even[j] = __builtin_amdgcn_perm(z, y, 0x05040100);
                    odd[j] = __builtin_amdgcn_perm(z, y, 0x07060302);
                }
                const auto e = __builtin_bit_cast(Half8<T>, even), f = __builtin_bit_cast(Half8<T>, odd);
                o[2 * i] = mma(e, lo, mma(e, hi, o[2 * i]));
                o[2 * i + 1] = mma(f, lo, mma(f, hi, o[2 * i + 1]));
            }
        }
        if (next < steps) x.v.load(a.c, x.row, lane);
    };
    for (int t = wave; t < steps; t += AHEAD * kWaves) {
#pragma unroll
        for (int u = 0; u < AHEAD; u++)
            if (t + u * kWaves < steps) compute(step[u], t + u * kWaves);
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // the waves' parts, joined in two rounds through LDS, register by register
    __shared__ float part[2][NT * 4 + 2][64];
#pragma unroll
    for (int half = kWaves / 2; half; half /= 2) {
        if (wave >= half && wave < 2 * half) {
            float(&to)[NT * 4 + 2][64] = part[wave - half];
#pragma unroll
            for (int i = 0; i < NT * 4; i++) to[i][lane] = o[i / 4][i % 4];
            to[NT * 4][lane] = m;
            to[NT * 4 + 1][lane] = l;
        }
        __syncthreads();
        if (wave < half) {
            const float(&in)[NT * 4 + 2][64] = part[wave];
            const float other = in[NT * 4][lane], both = fmaxf(m, other);
            const float x = exp2_of(m - or_zero(both)), y = exp2_of(other - or_zero(both));
            l = l * x + in[NT * 4 + 1][lane] * y;
#pragma unroll
            for (int i = 0; i < NT * 4; i++) o[i / 4][i % 4] = o[i / 4][i % 4] * x + in[i][lane] * y;
            m = both;
        }
        __syncthreads();
    }
    if (wave || !live) return;
    const bool alone = n <= a.chunk;
    if ((!alone || a.scores) && g == 0) a.sums[q_row * a.splits + split] = make_float2(m, l);
    if (alone) {
        const float x = l == 0.f ? 0.f : 1.f / l;
        T* to = static_cast<T*>(a.out) + q_row * D;
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) to[C::column(i, 4 * g + e)] = (T)(l == 0.f ? 0.f : o[i][e] * x);
    } else {
        float* to = a.parts + (q_row * a.splits + split) * D;
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) to[C::column(i, 4 * g + e)] = o[i][e];
    }
}

// What is left when all parts are there.  The first blocks join the parts of a
// query head each; the others add the weights of 1024 tokens of a kv head to
// their mass, from the scores that the first launch left.
constexpr int kMassKeys = 4 * kThreads;

// The largest reference and the sum over a query head's parts, by one wave.
__device__ __forceinline__ float2 total_of(const float2* sums, int parts, int lane) {
    float m = -__builtin_inff(), l = 0.f;
    for (int i = lane; i < parts; i += 64) m = fmaxf(m, sums[i].x);
    for (int x = 32; x; x /= 2) m = fmaxf(m, __shfl_xor(m, x));
    for (int i = lane; i < parts; i += 64) l += sums[i].y * exp2_of(sums[i].x - or_zero(m));
    for (int x = 32; x; x /= 2) l += __shfl_xor(l, x);
    return make_float2(or_zero(m), l);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) finish_kernel(Attend a, int joins) {
    __shared__ float4 sum[kThreads];
    __shared__ float2 total[kHeadTile * 16];
    const int lane = threadIdx.x & 63, dim = a.c.head_dim;
    if ((int)blockIdx.x < joins) {
        const int64_t q_row = blockIdx.x;
        const int n = length_of(a, (int)(q_row / a.q_heads));
        if (n <= a.chunk) return;
        const int parts = (n + a.chunk - 1) / a.chunk;
        const float2* sums = a.sums + q_row * a.splits;
        const float2 all = total_of(sums, parts, lane);
        const int wide = dim / 4, rows = kThreads / wide;  // four columns a thread
        const int r = threadIdx.x / wide, c = threadIdx.x % wide;
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < rows)
            for (int i = r; i < parts; i += rows) {
                const float w = exp2_of(sums[i].x - all.x);
                const float4 y = *reinterpret_cast<const float4*>(a.parts + (q_row * a.splits + i) * dim + 4 * c);
                x.x += w * y.x, x.y += w * y.y, x.z += w * y.z, x.w += w * y.w;
            }
        sum[threadIdx.x] = x;
        __syncthreads();
        if (r == 0) {
            for (int i = 1; i < rows; i++) {
                const float4 y = sum[i * wide + c];
                x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
            }
            const float f = all.y == 0.f ? 0.f : 1.f / all.y;
            T* to = static_cast<T*>(a.out) + q_row * dim + 4 * c;
            const float o[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; i++) to[i] = (T)(all.y == 0.f ? 0.f : o[i] * f);
        }
        return;
    }
    const int tiles = (a.bound + kMassKeys - 1) / kMassKeys;
    const int tile = (blockIdx.x - joins) % tiles, bh = (blockIdx.x - joins) / tiles;
    const int b = bh / a.c.kv_heads, h = bh % a.c.kv_heads;
    const int n = length_of(a, b);
    if (tile * kMassKeys >= n) return;
    const int parts = (n + a.chunk - 1) / a.chunk;
    const int64_t first = (int64_t)b * a.q_heads + h * a.group;
    const int key = tile * kMassKeys + 4 * threadIdx.x;
    vec<float, 4> w = {};
    for (int base = 0; base < a.group; base += kHeadTile * 16) {
        const int heads = min(a.group - base, kHeadTile * 16);
        __syncthreads();
        for (int i = threadIdx.x / 64; i < heads; i += kWaves) {
            const float2 t = total_of(a.sums + (first + base + i) * a.splits, parts, lane);
            if (lane == 0) total[i] = make_float2(t.x, t.y == 0.f ? 0.f : 1.f / t.y);
        }
        __syncthreads();
        if (key < n)
            for (int i = 0; i < heads; i++) {
                const auto s = *reinterpret_cast<const vec<float, 4>*>(a.scores + (first + base + i) * a.bound + key);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (total[i].y != 0.f) w[e] += exp2_of(s[e] - total[i].x) * total[i].y;
            }
    }
    if (key >= n) return;
    const int page = a.table[b * a.table_row + (key >> a.page_shift)];
    if (page < 0 || page >= a.c.pages) return;
    float* mass = a.c.mass + ((int64_t)page * a.c.kv_heads + h) * a.c.page_size + (key & (a.c.page_size - 1));
    for (int e = 0; e < 4; e++)
        if (key + e < n) unsafeAtomicAdd(mass + e, w[e]);
}

template <typename T, bool MX, int D>
int launch(const Attend& a, hipStream_t stream) {
    const int64_t groups = (int64_t)a.batch * a.c.kv_heads * a.head_tiles;
    hipLaunchKernelGGL((attend_kernel<T, MX, D>), dim3((unsigned)(groups * a.splits)), dim3(kThreads),
                       0, stream, a);
    if (const int rc = (int)hipGetLastError()) return rc;
    const int joins = a.splits > 1 ? a.batch * a.q_heads : 0;
    const int64_t tiles = a.scores ? (int64_t)((a.bound + kMassKeys - 1) / kMassKeys) * a.batch * a.c.kv_heads : 0;
    if (joins + tiles == 0) return 0;
    hipLaunchKernelGGL((finish_kernel<T>), dim3((unsigned)(joins + tiles)), dim3(kThreads), 0, stream, a, joins);
    return (int)hipGetLastError();
}

template <typename T, bool MX>
int attend(const Attend& a, hipStream_t stream) {
    switch (a.c.head_dim) {
        case 64: return launch<T, MX, 64>(a, stream);
        case 96: return launch<T, MX, 96>(a, stream);
        case 128: return launch<T, MX, 128>(a, stream);
        case 192: return launch<T, MX, 192>(a, stream);
        default: return launch<T, MX, 256>(a, stream);
    }
}

// How a call is split: enough parts to give every CU several workgroups, none
// shorter than a step of every wave.
constexpr int kWorkgroups = 256 * 8, kMinChunk = 128, kBestChunk = 1024;
struct Plan {
    int head_tiles, chunk, splits;
};
Plan plan(const vramc_kv_cache& c, int q_heads, int table_width, int batch) {
    Plan p;
    p.head_tiles = (q_heads / c.kv_heads + kHeadTile - 1) / kHeadTile;
    const int64_t bound = (int64_t)table_width * c.page_size;
    const int64_t groups = (int64_t)batch * c.kv_heads * p.head_tiles;
    int64_t chunk = bound * groups / kWorkgroups;
    chunk = (chunk + kMinChunk - 1) / kMinChunk * kMinChunk;
    if (chunk < kMinChunk) chunk = kMinChunk;
    if (chunk > kBestChunk) chunk = kBestChunk;
    p.chunk = (int)chunk;
    p.splits = (int)((bound + chunk - 1) / chunk);
    if (p.splits < 1) p.splits = 1;
    return p;
}

}  // namespace

extern "C" int64_t vramc_kv_attend_workspace(const vramc_kv_cache* c, int q_heads, int table_width,
                                             int batch, int track) {
    if (const int rc = check_cache(c)) return rc;
    if (q_heads <= 0 || q_heads % c->kv_heads || table_width < 0 || batch < 0) return RANS_EARG;
    const int64_t bound = (int64_t)table_width * c->page_size;
    if (bound > kMaxTokens || (int64_t)batch * q_heads > INT32_MAX / 2) return RANS_EARG;
    const Plan p = plan(*c, q_heads, table_width, batch);
    const int64_t rows = (int64_t)batch * q_heads;
    if (rows * p.splits > INT32_MAX / 2) return RANS_EARG;  // a grid's workgroups
    const int64_t parts = p.splits > 1 ? rows * p.splits * c->head_dim * 4 : 0;
    return parts + (track ? rows * bound * 4 : 0) + (track || parts ? rows * p.splits * 8 : 0);
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
    if (need && (!workspace || workspace_bytes < need)) return RANS_EWORKSPACE;
    if ((uintptr_t)workspace % 16) return RANS_EARG;
    const Plan p = plan(*c, q_heads, table_width, batch);
    const int64_t rows = (int64_t)batch * q_heads;
    Attend a{*c, q, q_seq, q_head, q_heads, q_heads / c->kv_heads, table, table_row, table_width,
             lengths, batch, scale, out, p.chunk, p.splits, p.head_tiles,
             __builtin_ctz(c->page_size), table_width * c->page_size, nullptr, nullptr, nullptr};
    auto* work = static_cast<float*>(workspace);
    if (p.splits > 1) {
        a.parts = work;
        work += rows * p.splits * c->head_dim;
    }
    if (track && table_width) {
        a.scores = work;
        work += rows * a.bound;
    }
    a.sums = reinterpret_cast<float2*>(work);
    if (c->dtype == RANS_X_F32) return attend<float, false>(a, stream);
    if (c->dtype == RANS_X_BF16)
        return c->mx ? attend<__bf16, true>(a, stream) : attend<__bf16, false>(a, stream);
    return c->mx ? attend<_Float16, true>(a, stream) : attend<_Float16, false>(a, stream);
}
