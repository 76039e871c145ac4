// Which pages of a sequence a query attends to: the smallest and largest key of each
// column of a page bound its scores, and those that can give the largest are taken.
//
// bound reads all keys of the pages once, and HBM bounds it: 2048 pages of 64 keys of 8
// heads of 128 columns 47.4 us, 5.8 TB/s of reads; 20.5 from 4 bits, whose conversion
// and comparisons keep the vectors busy.  A wave takes a page of a head; values are
// compared as whole numbers that sort as they do, two of 16 bits an instruction.
//
// select scores in 64 bits, so that a choice does not hang on the rounding of 32-bit
// sums.  Vector instructions bound it: 16 sequences of 512 pages of 8 heads, 5 query
// heads each, 16 us where their bounds are read in 6; the multiply-adds are a fifth of
// the instructions, the rest sums over lanes, conversions and addresses.  A second
// launch, a workgroup to a kv head of a sequence, finds the border by radix over the
// scores' bits, from the highest in which they differ, and writes the pages in their
// order by counts of ballot bits (5 to 7 us: reads, digits, lists, one after the other);
// for small tables it makes the scores too.
#include "kv_device.h"

#include <limits>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// ------------------------------------------------------------------ bounds
// Waves of a call: more entries, of a prompt's tokens most of which fill no page, are
// shared among them (one in 64 of 32768 entries of 8 heads 96 us with a wave to each).
constexpr int kBoundWaves = 1 << 14;

struct Bound {
    vramc_kv_cache c;
    int page_shift, lanes;    // lanes: of a row, a power of two
    const int32_t* pages;
    int64_t n;
    void* bounds;
    int64_t each;             // entries of the list to a wave
};

// Values as whole numbers that sort alike, and back: the bits below the sign are
// turned over in negative ones, two of 16 bits at once (which the compiler takes apart
// again unless it does not see where the signs come from).
template <typename I>
__device__ __forceinline__ vec<I, kPer> sorted(vec<I, kPer> x) {
    constexpr int N = kPer * sizeof(I) / 4;
    auto word = __builtin_bit_cast(vec<uint32_t, N>, x);
    const auto sign = __builtin_bit_cast(vec<uint32_t, N>, x >> (8 * sizeof(I) - 1));
#pragma unroll
    for (int i = 0; i < N; i++) {
        uint32_t turn = sign[i];
        asm("" : "+v"(turn));
        word[i] ^= turn & (sizeof(I) == 4 ? 0x7fffffffu : 0x7fff7fffu);
    }
    return __builtin_bit_cast(std::remove_reference_t<decltype(x)>, word);
}

// A lane's eight columns of a row.
template <typename T, bool MX>
struct Columns {
    using Int = std::conditional_t<sizeof(T) == 4, int32_t, int16_t>;
    using Whole = vec<Int, kPer>;
    static constexpr Int kInfinite = std::is_same_v<T, float> ? (Int)0x7f800000 : std::is_same_v<T, __bf16> ? 0x7f80 : 0x7c00;
    static constexpr Int kNaN = std::is_same_v<T, float> ? (Int)0x7fc00000 : std::is_same_v<T, __bf16> ? 0x7fc0 : 0x7e00;
    Lying<T> x;
    uint32_t codes, scale;
    // where a lane's first row begins, and rows that all lanes are further
    struct From {
        const Lying<T>* x;
        const uint32_t* codes;
        const uint8_t* scale;
        int per_row;
        __device__ __forceinline__ From(const vramc_kv_cache& c, int64_t row, int n, int seg) : per_row(n) {
            x = static_cast<const Lying<T>*>(c.k) + (row * n + seg);
            codes = static_cast<const uint32_t*>(c.k) + (row * n + seg);
            scale = c.k_scale + (row * (n / 4) + seg / 4);
        }
    };
    __device__ __forceinline__ void load(const From& from, int rows) {
        if constexpr (MX) {
            codes = from.codes[rows * from.per_row];
            scale = from.scale[rows * (from.per_row / 4)];
        } else {
            // past the caches, as nobody reads them next: 2048 pages of 64 keys of 8 heads
            // of 128 columns 48.6 us against 55.6
            const auto* at = from.x + rows * from.per_row;
#pragma unroll
            for (size_t i = 0; i < sizeof(T) / 2; i++) x.part[i] = __builtin_nontemporal_load(&at->part[i]);
        }
    }
    __device__ __forceinline__ Whole whole() const {
        if constexpr (MX) {
            vec<uint32_t, 4> pairs;
#pragma unroll
            for (int i = 0; i < 4; i++) pairs[i] = mx_pair_at<T>(codes, scale, i);
            return sorted<Int>(__builtin_bit_cast(Whole, pairs));
        } else {
            return sorted<Int>(__builtin_bit_cast(Whole, x));
        }
    }
};

template <typename V>
__device__ __forceinline__ V shuffled(V x, int d) {
    constexpr int N = sizeof(V) / 4;
    auto w = __builtin_bit_cast(vec<int, N>, x);
#pragma unroll
    for (int i = 0; i < N; i++) w[i] = __shfl_xor(w[i], d);
    return __builtin_bit_cast(V, w);
}

// AHEAD: loads of a wave under way, of which a page's steps are a multiple.
template <typename T, bool MX, int AHEAD>
__global__ void __launch_bounds__(kThreads) bound_kernel(Bound a) {
    using C = Columns<T, MX>;
    using Whole = typename C::Whole;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t chunk = blockIdx.x / a.c.kv_heads;
    const int head = blockIdx.x - chunk * a.c.kv_heads;
    const int per_row = a.c.head_dim / kPer, seg = lane & (a.lanes - 1), in_step = 64 / a.lanes;
    const int steps = a.c.page_size / in_step, first = lane / a.lanes;
    const bool inside = seg < per_row;
    // the wave's entries, up to 64 at once, and one page after the other of those that are
    const int64_t start = ((int64_t)chunk * kWaves + wave) * a.each, stop = min(start + a.each, a.n);
    for (int64_t i = start; i < stop; i += 64) {
        const int entry = i + lane < stop ? a.pages[i + lane] : -1;
        for (uint64_t some = __ballot((uint32_t)entry < (uint32_t)a.c.pages); some; some &= some - 1) {
            const int page = __builtin_amdgcn_readlane(entry, __builtin_ctzll(some));
            const int64_t at = (int64_t)page * a.c.kv_heads + head, row = (at << a.page_shift) + first;
            Whole low = std::numeric_limits<typename C::Int>::max(), high = std::numeric_limits<typename C::Int>::min();
            if (inside) {
                const typename C::From from(a.c, row, per_row, seg);
                for (int s = 0; s < steps; s += AHEAD) {
                    C x[AHEAD];
#pragma unroll
                    for (int u = 0; u < AHEAD; u++) x[u].load(from, (s + u) * in_step);
#pragma unroll
                    for (int u = 0; u < AHEAD; u++) {
                        const Whole y = x[u].whole();
                        low = __builtin_elementwise_min(low, y);
                        high = __builtin_elementwise_max(high, y);
                    }
                }
            }
            for (int d = a.lanes; d < 64; d *= 2) {
                low = __builtin_elementwise_min(low, shuffled(low, d));
                high = __builtin_elementwise_max(high, shuffled(high, d));
            }
            // what is not finite lies at or beyond the infinities
            const auto bad = (high >= C::kInfinite) | (low <= (typename C::Int)~C::kInfinite);
            if (inside && lane < 2 * a.lanes) {  // the first row's lanes write the smallest, the second's the largest
                const Whole y = bad ? (Whole)C::kNaN : sorted<typename C::Int>(lane < a.lanes ? low : high);
                static_cast<Lying<T>*>(a.bounds)[(2 * at + lane / a.lanes) * per_row + seg] = __builtin_bit_cast(Lying<T>, y);
            }
        }
    }
}

// ------------------------------------------------------------------ scores
// Query heads that vectors score; more the matrix cores, which take 16 as long as one.
// Both launches of 16 sequences of 512 pages, 8 heads of 128 columns: 16.9 us by vectors
// and 26.2 by matrices with one query head each, 23.3 and 26.6 with 5, 27.9 and 27.2 with
// 8, 41.1 and 29.5 with 16; heads of 64 columns meet at 8 too, of 256 beyond it.
constexpr int kFewHeads = 8;
constexpr int kSets = 2;          // of pages that a wave of vectors scores at once, a page to each row of lanes
constexpr int kMaxDim = 256;

struct Select {
    const void* bounds;
    const void* q;
    int64_t q_seq, q_head;
    int group, heads, pages, page_shift;
    const int32_t* table;
    int64_t table_row;
    int width;
    const int32_t* lengths;
    int batch, count, first, last;
    int chunks;                   // workgroups of a kv head of a sequence
    uint64_t* keys;               // [batch * heads][width]
    int32_t *chosen, *held;

    __device__ __forceinline__ int length_of(int b) const { return min(max(lengths[b], 0), width << page_shift); }
    __device__ __forceinline__ int pages_of(int n) const { return (n + (1 << page_shift) - 1) >> page_shift; }
    __device__ __forceinline__ int page(int b, int i) const {
        const int x = table[b * table_row + i];
        return (uint32_t)x < (uint32_t)pages ? x : -1;
    }
};

template <typename T>
__device__ __forceinline__ double wide(T x) {
    return (double)(float)x;
}

// The largest over 16 lanes.
__device__ __forceinline__ double row_max(double x) {
    const auto step = [&](auto control) {
        auto w = __builtin_bit_cast(vec<int, 2>, x);
#pragma unroll
        for (int i = 0; i < 2; i++) w[i] = __builtin_amdgcn_update_dpp(0, w[i], control(), 0xf, 0xf, true);
        x = fmax(x, __builtin_bit_cast(double, w));
    };
    step([] { return 0xb1; });   // quad_perm:[1,0,3,2]
    step([] { return 0x4e; });   // quad_perm:[2,3,0,1]
    step([] { return 0x141; });  // row_half_mirror
    step([] { return 0x140; });  // row_mirror
    return x;
}

// A page's score as a whole number that sorts alike; 0, below all, for no page.
__device__ __forceinline__ uint64_t key_of(double score, int page) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, score + 0.0);  // -0 as 0
    return page < 0 ? 0 : bits >> 63 ? ~bits : bits | 1ull << 63;
}

// The sum over the lanes of a row, 8 to 32.
__device__ __forceinline__ double row_sum(double x, int lanes) {
    const auto add = [&](auto control) {
        auto w = __builtin_bit_cast(vec<int, 2>, x);
#pragma unroll
        for (int i = 0; i < 2; i++) w[i] = __builtin_amdgcn_update_dpp(0, w[i], control(), 0xf, 0xf, true);
        x += __builtin_bit_cast(double, w);
    };
    add([] { return 0xb1; });   // quad_perm:[1,0,3,2]
    add([] { return 0x4e; });   // quad_perm:[2,3,0,1]
    add([] { return 0x141; });  // row_half_mirror
    if (lanes >= 16) add([] { return 0x140; });  // row_mirror
    if (lanes == 32) x += __shfl_xor(x, 16);
    return x;
}

// Few query heads: a wave scores two pages on each row of its lanes, eight columns a
// lane.  q_d lo_d or q_d hi_d is min(q_d, 0) lo_d + max(q_d, 0) hi_d, of which one is a
// zero: what a query does not point to leaves no rounding behind, so that pages alike
// where it points have the same score to the bit.
template <typename T>
struct Few {
    const Select& a;
    int b, h, dim, lanes, per_row, in_set, seg;
    bool inside;
    int page[kSets];
    Lying<T> raw[kSets][2];

    __device__ __forceinline__ Few(const Select& select, int sequence, int head, int d, int row_lanes)
        : a(select), b(sequence), h(head), dim(d), lanes(row_lanes), per_row(d / kPer), in_set(64 / row_lanes),
          seg(threadIdx.x & (row_lanes - 1)), inside(seg < d / kPer) {}
    // halves of the queries to LDS, [head][pair of eight][lane][2]
    __device__ __forceinline__ void stage(double* query, int threads) const {
        const T* q = static_cast<const T*>(a.q) + b * a.q_seq + (int64_t)h * a.group * a.q_head;
        for (int i = threadIdx.x; i < a.group * dim; i += threads) {
            const int g = i / dim, d = i - g * dim;
            query[((g * (kPer / 2) + d % kPer / 2) * per_row + d / kPer) * 2 + d % 2] = 0.5 * wide(q[g * a.q_head + d]);
        }
    }
    // the numbers of the lane's pages, from index `first` on, and their bounds
    __device__ __forceinline__ void find(int first) {
#pragma unroll
        for (int s = 0; s < kSets; s++) page[s] = a.page(b, min(first + s * in_set, a.width - 1));
    }
    __device__ __forceinline__ void load() {
#pragma unroll
        for (int s = 0; s < kSets; s++) {
            const auto* from = static_cast<const Lying<T>*>(a.bounds) +
                               2 * ((int64_t)max(page[s], 0) * a.heads + h) * per_row + (inside ? seg : 0);
#pragma unroll
            for (int i = 0; i < 2; i++) raw[s][i] = from[i * per_row];
        }
    }
    __device__ __forceinline__ void score(const double* query, double (&best)[kSets]) const {
        double low[kSets][kPer], high[kSets][kPer];
#pragma unroll
        for (int s = 0; s < kSets; s++) {
            const auto x = __builtin_bit_cast(vec<T, kPer>, raw[s][0]), y = __builtin_bit_cast(vec<T, kPer>, raw[s][1]);
#pragma unroll
            for (int j = 0; j < kPer; j++) low[s][j] = wide(x[j]), high[s][j] = wide(y[j]);
            best[s] = -__builtin_inf();
        }
        const int at = inside ? seg : 0;
#pragma unroll 1
        for (int g = 0; g < a.group; g++) {
            double x[kSets] = {}, y[kSets] = {};
#pragma unroll
            for (int p = 0; p < kPer / 2; p++) {
                const auto v = *reinterpret_cast<const vec<double, 2>*>(query + ((g * (kPer / 2) + p) * per_row + at) * 2);
#pragma unroll
                for (int i = 0; i < 2; i++) {  // of halves: the query's value or 0, exactly
                    const double below = v[i] - __builtin_fabs(v[i]), above = v[i] + __builtin_fabs(v[i]);
#pragma unroll
                    for (int s = 0; s < kSets; s++) {
                        x[s] = __builtin_fma(below, low[s][2 * p + i], x[s]);
                        y[s] = __builtin_fma(above, high[s][2 * p + i], y[s]);
                    }
                }
            }
#pragma unroll
            for (int s = 0; s < kSets; s++) {
                const double score = row_sum(inside ? x[s] + y[s] : 0.0, lanes);
                best[s] = score != score ? __builtin_inf() : fmax(best[s], score);
            }
        }
    }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) score_few_kernel(Select a, int dim, int lanes) {
    __shared__ __attribute__((aligned(16))) double query[kFewHeads * kMaxDim];
    const int group_of = blockIdx.x / a.chunks, chunk = blockIdx.x - group_of * a.chunks, b = group_of / a.heads;
    Few<T> few(a, b, group_of - b * a.heads, dim, lanes);
    const int wave = threadIdx.x >> 6, first = (chunk * kWaves + wave) * kSets * few.in_set + (threadIdx.x & 63) / lanes;
    few.find(first);  // while it is not known whether there are as many
    const int n = a.pages_of(a.length_of(b));
    if (n <= a.count || chunk * kWaves * kSets * few.in_set >= n) return;
    few.load();
    few.stage(query, kThreads);
    __syncthreads();
    double best[kSets];
    few.score(query, best);
#pragma unroll
    for (int s = 0; s < kSets; s++) {
        const int i = first + s * few.in_set;
        if (few.seg == 0 && i < n) a.keys[(int64_t)group_of * a.width + i] = key_of(best[s], few.page[s]);
    }
}

// A wave scores 16 pages with 16 query heads: lane (n = lane % 16, g = lane / 16)
// holds a quarter of the columns of page n's bounds, and reads those of head n from
// LDS.  Which columns a product takes from each quarter does not matter, as long as
// both sides take the same.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) score_kernel(Select a) {
    constexpr int QUARTER = D / 4, LOADS = QUARTER / kPer;
    __shared__ double query[D * 16];  // [column of a quarter][quarter][head]
    const int group_of = blockIdx.x / a.chunks, chunk = blockIdx.x - group_of * a.chunks;
    const int b = group_of / a.heads, h = group_of - b * a.heads;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const T* q = static_cast<const T*>(a.q) + b * a.q_seq + (int64_t)h * a.group * a.q_head;
    const auto stage = [&](int first) {  // zeros for heads that there are not
        for (int i = threadIdx.x; i < 16 * D; i += kThreads) {
            const int head = i / D, d = i % D;
            query[(d % QUARTER * 4 + d / QUARTER) * 16 + head] =
                first + head < a.group ? wide(q[(first + head) * a.q_head + d]) : 0.0;
        }
    };
    // the page's number and its bounds, while it is not known whether there are as many
    const int first = (chunk * kWaves + wave) * 16, page = a.page(b, min(first + (lane & 15), a.width - 1));
    const int n = a.pages_of(a.length_of(b));
    if (n <= a.count || chunk * kWaves * 16 >= n) return;
    Lying<T> low[LOADS], high[LOADS];
    const auto* from = static_cast<const Lying<T>*>(a.bounds) + ((int64_t)max(page, 0) * a.heads + h) * (2 * D / kPer) + g * LOADS;
#pragma unroll
    for (int i = 0; i < LOADS; i++) low[i] = from[i], high[i] = from[D / kPer + i];
    double best[4];
#pragma unroll
    for (int e = 0; e < 4; e++) best[e] = -__builtin_inf();
    for (int g0 = 0; g0 < a.group; g0 += 16) {
        if (g0) __syncthreads();
        stage(g0);
        __syncthreads();
        vec<double, 4> score = {};
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            const auto x = __builtin_bit_cast(vec<T, kPer>, low[i]), y = __builtin_bit_cast(vec<T, kPer>, high[i]);
#pragma unroll
            for (int j = 0; j < kPer; j++) {
                const double v = query[(i * kPer + j) * 64 + lane];
                score = __builtin_amdgcn_mfma_f64_16x16x4f64(wide(x[j]), v < 0 ? v : 0.0, score, 0, 0, 0);
                score = __builtin_amdgcn_mfma_f64_16x16x4f64(wide(y[j]), v < 0 ? 0.0 : v, score, 0, 0, 0);
            }
        }
        const bool live = g0 + (lane & 15) < a.group;
#pragma unroll
        for (int e = 0; e < 4; e++) {  // of page 4e + g
            const double s = score[e] != score[e] ? __builtin_inf() : score[e];
            best[e] = fmax(best[e], row_max(live ? s : -__builtin_inf()));
        }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int in = 4 * e + g;
        const int its = __shfl(page, in);
        if ((lane & 15) == e && first + in < n) a.keys[(int64_t)group_of * a.width + first + in] = key_of(best[e], its);
    }
}

// ------------------------------------------------------------------ choice
// Loops stay loops here: a workgroup waits for every line of its code (7.6 us with the
// keys in registers and everything unrolled, 6.0 so).
constexpr int kChoose = 512;                // threads
constexpr int kChooseWaves = kChoose / 64;
constexpr int kPiece = 4096;                // keys in LDS at once
// Small tables are scored where they are chosen from, by up to kFewHeads: so many pages
// at most, and as many as a workgroup scores in one step and a half.  16 sequences of 8
// heads of 128 columns, 5 query heads: 65 pages 9.2 us in one launch and 10.9 in two, 128
// 10.9 and 10.8, 256 17.0 and 14.0; of 2 heads of 64, 7 query heads, 128 8.5 and 10.2, 256
// 12.0 and 10.5.  Where the host waits, a launch and a workspace less are 4 us more.
constexpr int kHerePages = 192, kHereLanes = 1536;
constexpr int kDigit = 8, kBins = 1 << kDigit, kLaneBins = kBins / 64;  // 10 bits are fewer digits, and 1 us slower

__device__ __forceinline__ uint64_t from_bit(uint64_t x, int bit) { return bit < 64 ? x >> bit : 0; }

// HERE: the scores are made here, or else read.
template <typename T, bool HERE>
__global__ void __launch_bounds__(kChoose) choose_kernel(Select a, int dim, int lanes) {
    constexpr int PIECE = HERE ? kHerePages : kPiece, PARTS = PIECE / 64;  // keys at once, waves of them
    __shared__ uint64_t key[PIECE];
    __shared__ int32_t page[PIECE];
    // Every wave goes over the whole of what all have counted: one barrier a digit.
    __shared__ __attribute__((aligned(16))) int hist[3][kBins];  // this digit's, the last one's, the next one's
    __shared__ uint32_t ends[2][kChooseWaves];
    __shared__ uint32_t counts[PARTS];  // above the border | at it << 16
    const int b = blockIdx.x / a.heads, h = blockIdx.x - b * a.heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int32_t* out = a.chosen + (int64_t)blockIdx.x * a.count;
    const auto entry = [&](int i) {
        const int page = a.page(b, i);
        return page < 0 ? -1 : page * a.heads + h;
    };
    const uint64_t* keys = a.keys + (int64_t)blockIdx.x * a.width + a.first;
    const auto load = [&](int piece, int size) {  // a thread reads what it wrote
#pragma unroll 2
        for (int i = threadIdx.x; i < size; i += kChoose) {
            const uint64_t x = keys[piece * PIECE + i];
            const int32_t y = entry(a.first + piece * PIECE + i);
            key[i] = x, page[i] = y;
        }
    };
    // the first keys, while it is not known how many there are
    if (!HERE && a.width > a.count) load(0, min(a.width - a.first, PIECE));
    const int tokens = a.length_of(b), n = a.pages_of(tokens), kept = min(n, a.count);
    if (threadIdx.x == 0) a.held[blockIdx.x] = kept ? tokens - ((n - kept) << a.page_shift) : 0;
    // the pages at the ends, or all of them, and what is behind them
    const int left = n <= a.count ? n : a.first, right = n <= a.count ? 0 : a.last;
#pragma unroll 1
    for (int i = threadIdx.x; i < a.count; i += kChoose)
        if (i < left || i >= a.count - right || i >= kept)
            out[i] = i < left ? entry(i) : i >= kept ? -1 : entry(n - a.count + i);
    const int among = n - a.first - a.last;      // candidates,
    int room = a.count - a.first - a.last;       // of which so many are taken
    if (n <= a.count || room == 0) return;
    const int pieces = HERE ? 1 : (among + PIECE - 1) / PIECE;
    const auto size_of = [&](int piece) { return min(among - piece * PIECE, PIECE); };
    if constexpr (HERE) {
        __shared__ __attribute__((aligned(16))) double query[kFewHeads * kMaxDim];
        Few<T> few(a, b, h, dim, lanes);
        const int step = kSets * few.in_set;  // of a wave
        int first = wave * step + lane / lanes;
        few.find(first);
        few.load();
        few.stage(query, kChoose);
        __syncthreads();
#pragma unroll 1
        for (; first - lane / lanes < n; first += kChooseWaves * step) {
            double best[kSets];
            few.score(query, best);
#pragma unroll
            for (int s = 0; s < kSets; s++) {
                const int i = first + s * few.in_set - a.first;
                if (few.seg == 0 && i >= 0 && i < among) {
                    key[i] = key_of(best[s], few.page[s]);
                    page[i] = few.page[s] < 0 ? -1 : few.page[s] * a.heads + h;
                }
            }
            few.find(first + kChooseWaves * step);
            few.load();
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < 3 * kBins; i += kChoose) (&hist[0][0])[i] = 0;
    // the highest of the upper 32 bits in which keys differ, or the 32nd
    uint32_t least = ~0u, most = 0;
#pragma unroll 1
    for (int piece = 0; piece < pieces; piece++) {
        if (piece) load(piece, size_of(piece));
#pragma unroll 1
        for (int i = threadIdx.x; i < size_of(piece); i += kChoose) {
            const uint32_t x = (uint32_t)(key[i] >> 32);
            least = min(least, x), most = max(most, x);
        }
    }
#pragma unroll
    for (int d = 32; d; d /= 2) {
        least = min(least, (uint32_t)__shfl_xor((int)least, d));
        most = max(most, (uint32_t)__shfl_xor((int)most, d));
    }
    if (lane == 0) ends[0][wave] = least, ends[1][wave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kChooseWaves; w++) least = min(least, ends[0][w]), most = max(most, ends[1][w]);
    int bit = least == most ? 32 : 64 - __builtin_clz(least ^ most);
    uint64_t above = bit < 64 ? (uint64_t)most >> (bit - 32) : 0;  // what the border's keys have from that bit on
    int at = among;                                                // how many keys have it
#pragma unroll 1
    for (int turn = 0; bit > 0 && at > room; turn = turn == 2 ? 0 : turn + 1) {
        const int digit = min(bit, kDigit), low = bit - digit, bins = 1 << digit;
#pragma unroll 1
        for (int piece = 0; piece < pieces; piece++) {
            if (pieces > 1) load(piece, size_of(piece));
#pragma unroll 1
            for (int i = threadIdx.x; i < size_of(piece); i += kChoose) {
                const uint64_t x = key[i];
                if (from_bit(x, bit) == above) atomicAdd(&hist[turn][x >> low & (bins - 1)], 1);
            }
        }
        __syncthreads();
        // the last digit's bins, which all have read now, for the digit behind the next
        for (int i = threadIdx.x; i < kBins; i += kChoose) hist[turn == 0 ? 2 : turn - 1][i] = 0;
        // the bin that holds the room-th from the top, neighbouring bins to a lane
        int x[kLaneBins], sum = 0;
#pragma unroll
        for (int i = 0; i < kLaneBins; i += 4) {
            const auto y = *reinterpret_cast<const vec<int, 4>*>(&hist[turn][(63 - lane) * kLaneBins + i]);
#pragma unroll
            for (int j = 0; j < 4; j++) sum += x[i + j] = y[j];
        }
        int before = wave_scan(sum) - sum;
        const int owner = __builtin_ctzll(__ballot(before < room && before + sum >= room));
        int bin = 0, count = 0;
        bool found = false;
#pragma unroll
        for (int i = kLaneBins - 1; i >= 0; i--) {
            const bool it = !found && before + x[i] >= room;
            if (it) bin = (63 - lane) * kLaneBins + i, count = x[i];
            found |= it;
            if (!found) before += x[i];
        }
        bin = __builtin_amdgcn_readlane(bin, owner);
        room -= __builtin_amdgcn_readlane(before, owner);
        at = __builtin_amdgcn_readlane(count, owner);
        above = above << digit | (uint64_t)bin;
        bit = low;
    }
    // those above the border, and the first `room` of those at it, in their order
    uint32_t taken = 0, equal = 0;  // of the pieces before
#pragma unroll 1
    for (int piece = 0; piece < pieces; piece++) {
        const int size = size_of(piece), parts = (size + 63) / 64;
        if (pieces > 1) {
            load(piece, size_of(piece));
            __syncthreads();  // the last piece's counts have been read
        }
#pragma unroll 1
        for (int i = threadIdx.x; i - lane < size; i += kChoose) {
            const uint64_t x = i < size ? from_bit(key[i], bit) : 0;
            const uint32_t more = __popcll(__ballot(i < size && x > above)), same = __popcll(__ballot(i < size && x == above));
            if (lane == 0) counts[i / 64] = more | same << 16;
        }
        __syncthreads();
        const uint32_t mine = lane < parts ? counts[lane] : 0, sum = (uint32_t)wave_scan((int)mine);
#pragma unroll 1
        for (int i = threadIdx.x; i - lane < size; i += kChoose) {
            const uint64_t x = i < size ? from_bit(key[i], bit) : 0;
            const uint64_t more = __ballot(i < size && x > above), same = __ballot(i < size && x == above);
            const uint32_t before = (uint32_t)__builtin_amdgcn_readlane((int)(sum - mine), (i - lane) / 64);
            const auto below = [&](uint64_t mask) {
                return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
            };
            const uint32_t like = equal + (before >> 16) + below(same);
            if (i < size && (x > above || (x == above && like < (uint32_t)room)))
                out[a.first + taken + (before & 0xffff) + below(more) + min(like, (uint32_t)room)] = page[i];
        }
        const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
        taken += all & 0xffff;
        equal += all >> 16;
    }
}

int lanes_of(int dim) { return dim <= 64 ? 8 : dim <= 128 ? 16 : 32; }

// Workgroups that score a row of the table.
int64_t chunks_of(int dim, int group, int table_width) {
    const int pages = group <= kFewHeads ? kWaves * kSets * 64 / lanes_of(dim) : kWaves * 16;
    return (table_width + pages - 1) / pages;
}

// Whether the workgroups that choose make the scores themselves.
bool scored_here(int dim, int group, int table_width) {
    return group <= kFewHeads && (int64_t)table_width * lanes_of(dim) <= kHereLanes;
}

template <typename T>
int select(const Select& a, int dim, hipStream_t stream) {
    const int lanes = lanes_of(dim);
    const dim3 chosen((unsigned)(a.batch * a.heads)), choose(kChoose);
    if (a.width > a.count && scored_here(dim, a.group, a.width)) {
        hipLaunchKernelGGL((choose_kernel<T, true>), chosen, choose, 0, stream, a, dim, lanes);
        return (int)hipGetLastError();
    }
    if (a.width > a.count) {
        const dim3 grid((unsigned)((int64_t)a.batch * a.heads * a.chunks)), block(kThreads);
        if (a.group <= kFewHeads) hipLaunchKernelGGL((score_few_kernel<T>), grid, block, 0, stream, a, dim, lanes);
        else if (dim == 64) hipLaunchKernelGGL((score_kernel<T, 64>), grid, block, 0, stream, a);
        else if (dim == 96) hipLaunchKernelGGL((score_kernel<T, 96>), grid, block, 0, stream, a);
        else if (dim == 128) hipLaunchKernelGGL((score_kernel<T, 128>), grid, block, 0, stream, a);
        else if (dim == 192) hipLaunchKernelGGL((score_kernel<T, 192>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((score_kernel<T, 256>), grid, block, 0, stream, a);
        if (const int rc = (int)hipGetLastError()) return rc;
    }
    hipLaunchKernelGGL((choose_kernel<float, false>), chosen, choose, 0, stream, a, dim, lanes);  // of any type
    return (int)hipGetLastError();
}

template <typename T, bool MX>
int bound(const Bound& a, hipStream_t stream) {
    const int64_t blocks = (a.n + kWaves * a.each - 1) / (kWaves * a.each) * a.c.kv_heads;
    if (blocks > kMaxThreads / kThreads) return RANS_EARG;
    const dim3 grid((unsigned)blocks), block(kThreads);
    const int steps = a.c.page_size * a.lanes / 64;
    // four rows of f32 fill as many registers as eight of 16 bits (108 us against 126), and
    // 4-bit ones are bound by their conversion (20.5 us against 21.7)
    constexpr bool EIGHT = sizeof(T) == 2 && !MX;
    if (steps >= 8 && EIGHT) hipLaunchKernelGGL((bound_kernel<T, MX, EIGHT ? 8 : 4>), grid, block, 0, stream, a);
    else if (steps >= 4) hipLaunchKernelGGL((bound_kernel<T, MX, 4>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((bound_kernel<T, MX, 2>), grid, block, 0, stream, a);
    return (int)hipGetLastError();
}

Span span_of_bounds(const vramc_kv_cache& c, const void* bounds) {
    return {bounds, head_pages(c) * 2 * c.head_dim * (c.dtype == RANS_X_F32 ? 4 : 2)};
}

}  // namespace

extern "C" int vramc_kv_bound(const vramc_kv_cache* c, const int32_t* pages, int64_t n, void* bounds,
                              hipStream_t stream) {
    if (const int rc = check_cache(c)) return rc;
    if (n < 0 || n > INT64_MAX / 65536) return RANS_EARG;
    if (n == 0) return 0;
    if (!pages || !bounds || (uintptr_t)bounds % 16) return RANS_EARG;
    // Waves read these while others write.
    const Span out[] = {span_of_bounds(*c, bounds)};
    if (overlap(out[0], Span{pages, n * 4}) || overlap(out, spans_of(*c).of)) return RANS_EARG;
    const Bound a{*c, __builtin_ctz(c->page_size), lanes_of(c->head_dim), pages, n, bounds,
                  (n * c->kv_heads + kBoundWaves - 1) / kBoundWaves};
    if (c->dtype == RANS_X_F32) return bound<float, false>(a, stream);
    if (c->dtype == RANS_X_BF16) return c->mx ? bound<__bf16, true>(a, stream) : bound<__bf16, false>(a, stream);
    return c->mx ? bound<_Float16, true>(a, stream) : bound<_Float16, false>(a, stream);
}

extern "C" int64_t vramc_kv_select_workspace(const vramc_kv_cache* c, int q_heads, int table_width, int batch, int count) {
    if (const int rc = check_cache(c)) return rc;
    if (q_heads <= 0 || q_heads % c->kv_heads || table_width < 0 || batch < 0 || count <= 0 ||
        (int64_t)table_width * c->page_size > kMaxTokens || (int64_t)batch * c->kv_heads > kMaxThreads / kChoose ||
        (int64_t)count * c->page_size > kMaxTokens || (int64_t)c->pages * c->kv_heads > INT32_MAX)
        return RANS_EARG;
    const int group = q_heads / c->kv_heads;
    if (table_width <= count || scored_here(c->head_dim, group, table_width)) return 0;
    const int64_t rows = (int64_t)batch * c->kv_heads;
    if (chunks_of(c->head_dim, group, table_width) * rows > kMaxThreads / kThreads) return RANS_EARG;
    return rows * table_width * 8;
}

extern "C" int vramc_kv_select(const vramc_kv_cache* c, const void* bounds, const void* q, int64_t q_seq,
                               int64_t q_head, int q_heads, const int32_t* table, int64_t table_row,
                               int table_width, const int32_t* lengths, int batch, int count, int first,
                               int last, int32_t* chosen, int32_t* held, void* workspace,
                               int64_t workspace_bytes, hipStream_t stream) {
    const int64_t need = vramc_kv_select_workspace(c, q_heads, table_width, batch, count);
    if (need < 0) return (int)need;
    if (first < 0 || last < 1 || (int64_t)first + last > count) return RANS_EARG;
    if (batch == 0) return 0;
    if (!bounds || (uintptr_t)bounds % 16 || !q || !lengths || !chosen || !held || (table_width && !table))
        return RANS_EARG;
    if (need && (!workspace || workspace_bytes < need)) return RANS_EWORKSPACE;
    if (need && (uintptr_t)workspace % 16) return RANS_EARG;
    // Workgroups read these while others write.
    const int64_t rows = (int64_t)batch * c->kv_heads;
    const Span out[] = {{chosen, rows * count * 4}, {held, rows * 4}, {workspace, need}};
    const Span read[] = {
        span_of_bounds(*c, bounds), {lengths, batch * (int64_t)4}, span_of(table, table_row, 0, batch, 1, table_width, 4),
        span_of(q, q_seq, q_head, batch, q_heads, c->head_dim, c->dtype == RANS_X_F32 ? 4 : 2)};
    if (overlap(out, read) || overlap(out[0], out[1]) || overlap(out[0], out[2]) || overlap(out[1], out[2]))
        return RANS_EARG;
    const Select a{bounds, q, q_seq, q_head, q_heads / c->kv_heads, c->kv_heads, c->pages,
                   __builtin_ctz(c->page_size), table, table_row, table_width, lengths, batch, count, first, last,
                   (int)chunks_of(c->head_dim, q_heads / c->kv_heads, table_width), static_cast<uint64_t*>(workspace), chosen, held};
    if (c->dtype == RANS_X_F32) return select<float>(a, c->head_dim, stream);
    return c->dtype == RANS_X_BF16 ? select<__bf16>(a, c->head_dim, stream) : select<_Float16>(a, c->head_dim, stream);
}
