// Which pages of a sequence a query attends to: the smallest and largest key of each
// column of a page bound its scores, and those that can give the largest are taken.
//
// bound reads all keys of the pages once, and HBM bounds it.  A wave takes a page of
// a head; values are compared as whole numbers that sort as they do, two of 16 bits
// an instruction.
//
// select reads two rows a page and head, q_d lo_d or q_d hi_d being q_d mid_d +
// |q_d| half_d whatever the sign: two multiply-adds a column and query head, in 64
// bits, which MI355X makes at the rate of 32, so that which page is taken does not
// depend on an order of sums.  A second launch, a workgroup to a kv head of a
// sequence, finds the border by radix over the scores' bits, from the highest in
// which they differ, and writes the pages in their order by counts of ballot bits.
#include "kv_device.h"

#include <limits>

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// ------------------------------------------------------------------ bounds
constexpr int kEntries = 16;  // of the list, to a workgroup
constexpr int kAhead = 8;     // loads of a wave under way

struct Bound {
    vramc_kv_cache c;
    int page_shift, lanes;    // lanes: of a row, a power of two
    const int32_t* pages;
    int64_t n;
    void* bounds;
};

// Values as whole numbers that sort alike, and back: the bits below the sign are
// turned over in negative ones.
template <typename I>
__device__ __forceinline__ vec<I, kPer> sorted(vec<I, kPer> x) {
    return x ^ ((x >> (8 * sizeof(I) - 1)) & std::numeric_limits<I>::max());
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
    __device__ __forceinline__ void load(const vramc_kv_cache& c, int64_t row, int per_row, int seg) {
        if constexpr (MX) {
            codes = static_cast<const uint32_t*>(c.k)[row * per_row + seg];
            scale = c.k_scale[row * (per_row / 4) + seg / 4];
        } else {
            x = static_cast<const Lying<T>*>(c.k)[row * per_row + seg];
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

template <typename T, bool MX>
__global__ void __launch_bounds__(kThreads) bound_kernel(Bound a) {
    using C = Columns<T, MX>;
    using Whole = typename C::Whole;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t chunk = blockIdx.x / a.c.kv_heads;
    const int head = blockIdx.x - chunk * a.c.kv_heads;
    const int per_row = a.c.head_dim / kPer, seg = lane & (a.lanes - 1), in_step = 64 / a.lanes;
    const int steps = a.c.page_size / in_step, first = lane / a.lanes;
    const bool inside = seg < per_row;
    for (int e = 0; e < kEntries / kWaves; e++) {
        const int64_t i = (int64_t)chunk * kEntries + e * kWaves + wave;
        const int page = i < a.n ? a.pages[i] : -1;
        if (page < 0 || page >= a.c.pages) continue;
        const int64_t at = (int64_t)page * a.c.kv_heads + head, row = (at << a.page_shift) + first;
        Whole low = std::numeric_limits<typename C::Int>::max(), high = std::numeric_limits<typename C::Int>::min();
        for (int s = 0; s < steps; s += kAhead) {
            C x[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; u++)  // beyond the last step the last again
                if (inside) x[u].load(a.c, row + (int64_t)min(s + u, steps - 1) * in_step, per_row, seg);
#pragma unroll
            for (int u = 0; u < kAhead; u++)
                if (inside) {
                    const Whole y = x[u].whole();
                    low = __builtin_elementwise_min(low, y);
                    high = __builtin_elementwise_max(high, y);
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

// ------------------------------------------------------------------ scores
constexpr int kSets = 2;          // of pages that a wave scores at once, a page to each row of lanes
constexpr int kHeads = 16;        // query heads in LDS at once
constexpr int kMaxDim = 256;

struct Select {
    const void* bounds;
    const void* q;
    int64_t q_seq, q_head;
    int group, heads, dim, lanes, pages, page_shift;
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

template <typename T>
__global__ void __launch_bounds__(kThreads) score_kernel(Select a) {
    __shared__ __attribute__((aligned(16))) double query[kHeads * kMaxDim];  // [head][pair of eight][lane][2]
    const int group_of = blockIdx.x / a.chunks, chunk = blockIdx.x - group_of * a.chunks;
    const int b = group_of / a.heads, h = group_of - b * a.heads;
    const int n = a.pages_of(a.length_of(b));
    const int in_set = 64 / a.lanes, start = chunk * (kWaves * kSets * in_set);
    if (n <= a.count || start >= n) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int per_row = a.dim / kPer, seg = lane & (a.lanes - 1);
    const bool inside = seg < per_row;
    int index[kSets], page[kSets];
    Lying<T> raw[kSets][2];
#pragma unroll
    for (int s = 0; s < kSets; s++) {
        index[s] = start + (wave * kSets + s) * in_set + lane / a.lanes;
        page[s] = index[s] < n ? a.page(b, index[s]) : -1;
    }
#pragma unroll
    for (int s = 0; s < kSets; s++) {
        const auto* from = static_cast<const Lying<T>*>(a.bounds) + 2 * ((int64_t)max(page[s], 0) * a.heads + h) * per_row + seg;
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (inside) raw[s][i] = from[i * per_row];
            else raw[s][i] = {};
    }
    double middle[kSets][kPer], half[kSets][kPer], best[kSets];
#pragma unroll
    for (int s = 0; s < kSets; s++) {
        const auto low = __builtin_bit_cast(vec<T, kPer>, raw[s][0]), high = __builtin_bit_cast(vec<T, kPer>, raw[s][1]);
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            middle[s][j] = 0.5 * (wide(high[j]) + wide(low[j]));
            half[s][j] = 0.5 * (wide(high[j]) - wide(low[j]));
        }
        best[s] = -__builtin_inf();
    }
    const int at = seg < per_row ? seg : 0;
    for (int g0 = 0; g0 < a.group; g0 += kHeads) {
        const int heads = min(kHeads, a.group - g0);
        const T* q = static_cast<const T*>(a.q) + b * a.q_seq + (int64_t)(h * a.group + g0) * a.q_head;
        if (g0) __syncthreads();
        for (int i = threadIdx.x; i < heads * a.dim; i += kThreads) {
            const int g = i / a.dim, d = i - g * a.dim;
            query[((g * (kPer / 2) + d % kPer / 2) * per_row + d / kPer) * 2 + d % 2] = wide(q[g * a.q_head + d]);
        }
        __syncthreads();
        for (int g = 0; g < heads; g++) {
            double x[kSets] = {}, y[kSets] = {};
#pragma unroll
            for (int p = 0; p < kPer / 2; p++) {
                const auto v = *reinterpret_cast<const vec<double, 2>*>(query + ((g * (kPer / 2) + p) * per_row + at) * 2);
#pragma unroll
                for (int s = 0; s < kSets; s++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        x[s] = __builtin_fma(v[i], middle[s][2 * p + i], x[s]);
                        y[s] = __builtin_fma(__builtin_fabs(v[i]), half[s][2 * p + i], y[s]);
                    }
            }
#pragma unroll
            for (int s = 0; s < kSets; s++) {
                const double score = row_sum(inside ? x[s] + y[s] : 0.0, a.lanes);
                best[s] = score != score ? __builtin_inf() : fmax(best[s], score);
            }
        }
    }
#pragma unroll
    for (int s = 0; s < kSets; s++)
        if (seg == 0 && index[s] < n) {  // 0 for no page: below all scores
            const uint64_t bits = __builtin_bit_cast(uint64_t, best[s] + 0.0);  // -0 as 0
            const uint64_t key = bits >> 63 ? ~bits : bits | 1ull << 63;
            a.keys[(int64_t)group_of * a.width + index[s]] = page[s] < 0 ? 0 : key;
        }
}

// ------------------------------------------------------------------ choice
constexpr int kChoose = 512;                // threads
constexpr int kChooseWaves = kChoose / 64;
constexpr int kKeys = 16;                   // keys of a thread
constexpr int kPiece = kChoose * kKeys;
constexpr int kDigit = 10, kBins = 1 << kDigit;

__device__ __forceinline__ uint64_t from_bit(uint64_t x, int bit) { return bit < 64 ? x >> bit : 0; }

__global__ void __launch_bounds__(kChoose) choose_kernel(Select a) {
    __shared__ int hist[kBins], found[3], waves[kChooseWaves];
    __shared__ uint64_t ends[2][kChooseWaves];
    __shared__ uint32_t counts[kKeys * kChooseWaves];  // above the border | at it << 16
    __shared__ uint32_t sums[kKeys * kChooseWaves];
    const int b = blockIdx.x / a.heads, h = blockIdx.x - b * a.heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tokens = a.length_of(b), n = a.pages_of(tokens), kept = min(n, a.count);
    int32_t* out = a.chosen + (int64_t)blockIdx.x * a.count;
    const auto entry = [&](int i) {
        const int page = a.page(b, i);
        return page < 0 ? -1 : page * a.heads + h;
    };
    if (threadIdx.x == 0) a.held[blockIdx.x] = kept ? tokens - ((n - kept) << a.page_shift) : 0;
    for (int i = kept + threadIdx.x; i < a.count; i += kChoose) out[i] = -1;
    if (n <= a.count) {
        for (int i = threadIdx.x; i < n; i += kChoose) out[i] = entry(i);
        return;
    }
    for (int i = threadIdx.x; i < a.first; i += kChoose) out[i] = entry(i);
    for (int i = threadIdx.x; i < a.last; i += kChoose) out[a.count - a.last + i] = entry(n - a.last + i);
    const int among = n - a.first - a.last;      // candidates,
    int room = a.count - a.first - a.last;       // of which so many are taken
    if (room == 0) return;
    const uint64_t* keys = a.keys + (int64_t)blockIdx.x * a.width + a.first;
    const int pieces = (among + kPiece - 1) / kPiece;
    uint64_t key[kKeys];
    const auto there = [&](int piece, int u) { return piece * kPiece + u * kChoose + (int)threadIdx.x < among; };
    const auto load = [&](int piece) {
#pragma unroll
        for (int u = 0; u < kKeys; u++)
            if (there(piece, u)) key[u] = keys[piece * kPiece + u * kChoose + threadIdx.x];
    };
    // f(u, key, whether it is one) over a piece's keys, the same for all threads of a wave
    const auto over = [&](int piece, auto f) {
#pragma unroll
        for (int u = 0; u < kKeys; u++)
            if (piece * kPiece + u * kChoose < among) f(u, key[u], there(piece, u));
    };
    // the highest bit in which keys differ
    uint64_t least = ~0ull, most = 0;
    for (int piece = 0; piece < pieces; piece++) {
        load(piece);
        over(piece, [&](int, uint64_t k, bool is) {
            if (is) least = min(least, k), most = max(most, k);
        });
    }
#pragma unroll
    for (int d = 32; d; d /= 2) {
        least = min(least, (uint64_t)__shfl_xor((unsigned long long)least, d));
        most = max(most, (uint64_t)__shfl_xor((unsigned long long)most, d));
    }
    if (lane == 0) ends[0][wave] = least, ends[1][wave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kChooseWaves; w++) least = min(least, ends[0][w]), most = max(most, ends[1][w]);
    int bit = least == most ? 0 : 64 - __builtin_clzll(least ^ most);
    uint64_t above = from_bit(most, bit);  // what the border's keys have from that bit on
    int at = among;                        // how many keys have it
    while (bit > 0 && at > room) {
        const int digit = min(bit, kDigit), low = bit - digit, bins = 1 << digit;
        for (int i = threadIdx.x; i < kBins; i += kChoose) hist[i] = 0;
        __syncthreads();
        for (int piece = 0; piece < pieces; piece++) {
            if (pieces > 1) load(piece);
            over(piece, [&](int, uint64_t k, bool is) {
                if (is && from_bit(k, bit) == above) atomicAdd(&hist[k >> low & (bins - 1)], 1);
            });
        }
        __syncthreads();
        // from the top, two bins to a thread
        const int top = bins - 1 - 2 * (int)threadIdx.x;
        const int x = top >= 0 ? hist[top] : 0, y = top >= 1 ? hist[top - 1] : 0, both = wave_scan(x + y);
        if (lane == 63) waves[wave] = both;
        __syncthreads();
        int before = both - x - y;
#pragma unroll
        for (int w = 0; w < kChooseWaves; w++) before += w < wave ? waves[w] : 0;
        if (before < room && before + x + y >= room) {
            const bool second = before + x < room;
            found[0] = second ? top - 1 : top;
            found[1] = second ? before + x : before;
            found[2] = second ? y : x;
        }
        __syncthreads();
        above = above << digit | (uint64_t)found[0];
        room -= found[1];
        at = found[2];
        bit = low;
    }
    // those above the border, and the first `room` of those at it, in their order
    uint32_t taken = 0;  // of the pieces before, packed alike
    uint32_t equal = 0;
    for (int piece = 0; piece < pieces; piece++) {
        if (pieces > 1) load(piece);
        __syncthreads();
        over(piece, [&](int u, uint64_t k, bool is) {
            const uint64_t x = from_bit(k, bit);
            const uint32_t more = __popcll(__ballot(is && x > above)), same = __popcll(__ballot(is && x == above));
            if (lane == 0) counts[u * kChooseWaves + wave] = more | same << 16;
        });
        __syncthreads();
        const int parts = min(kKeys, (among - piece * kPiece + kChoose - 1) / kChoose) * kChooseWaves;
        if (wave == 0) {  // two of them to a lane
            const uint32_t x = 2 * lane < parts ? counts[2 * lane] : 0, y = 2 * lane + 1 < parts ? counts[2 * lane + 1] : 0;
            const uint32_t sum = (uint32_t)wave_scan((int)(x + y));
            sums[2 * lane] = sum - y;
            sums[2 * lane + 1] = sum;
        }
        __syncthreads();
        over(piece, [&](int u, uint64_t k, bool is) {
            const uint64_t x = from_bit(k, bit);
            const uint64_t more = __ballot(is && x > above), same = __ballot(is && x == above);
            const int i = u * kChooseWaves + wave;
            const uint32_t before = sums[i] - counts[i];
            const auto below = [&](uint64_t mask) {
                return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
            };
            const uint32_t like = equal + (before >> 16) + below(same);
            if (is && (x > above || (x == above && like < (uint32_t)room)))
                out[a.first + taken + (before & 0xffff) + below(more) + min(like, (uint32_t)room)] =
                    entry(a.first + piece * kPiece + u * kChoose + threadIdx.x);
        });
        const uint32_t last = sums[parts - 1];
        taken += last & 0xffff;
        equal += last >> 16;
    }
}

int lanes_of(int dim) { return dim <= 64 ? 8 : dim <= 128 ? 16 : 32; }

template <typename T, bool MX>
int bound(const Bound& a, hipStream_t stream) {
    const int64_t blocks = (a.n + kEntries - 1) / kEntries * a.c.kv_heads;
    if (blocks > kMaxThreads / kThreads) return RANS_EARG;
    hipLaunchKernelGGL((bound_kernel<T, MX>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, a);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" int vramc_kv_bound(const vramc_kv_cache* c, const int32_t* pages, int64_t n, void* bounds,
                              hipStream_t stream) {
    if (const int rc = check_cache(c)) return rc;
    if (n < 0 || n > INT64_MAX / 65536) return RANS_EARG;
    if (n == 0) return 0;
    if (!pages || !bounds || (uintptr_t)bounds % 16) return RANS_EARG;
    const Bound a{*c, __builtin_ctz(c->page_size), lanes_of(c->head_dim), pages, n, bounds};
    if (c->dtype == RANS_X_F32) return bound<float, false>(a, stream);
    if (c->dtype == RANS_X_BF16) return c->mx ? bound<__bf16, true>(a, stream) : bound<__bf16, false>(a, stream);
    return c->mx ? bound<_Float16, true>(a, stream) : bound<_Float16, false>(a, stream);
}

extern "C" int64_t vramc_kv_select_workspace(const vramc_kv_cache* c, int table_width, int batch, int count) {
    if (const int rc = check_cache(c)) return rc;
    if (table_width < 0 || batch < 0 || count <= 0 || (int64_t)table_width * c->page_size > kMaxTokens ||
        (int64_t)batch * c->kv_heads > kMaxThreads / kChoose || (int64_t)count * c->page_size > kMaxTokens ||
        (int64_t)c->pages * c->kv_heads > INT32_MAX)
        return RANS_EARG;
    if (table_width <= count) return 0;
    const int in_block = kWaves * kSets * 64 / lanes_of(c->head_dim);
    const int64_t chunks = (table_width + in_block - 1) / in_block, rows = (int64_t)batch * c->kv_heads;
    if (chunks * rows > kMaxThreads / kThreads) return RANS_EARG;
    return rows * table_width * 8;
}

extern "C" int vramc_kv_select(const vramc_kv_cache* c, const void* bounds, const void* q, int64_t q_seq,
                               int64_t q_head, int q_heads, const int32_t* table, int64_t table_row,
                               int table_width, const int32_t* lengths, int batch, int count, int first,
                               int last, int32_t* chosen, int32_t* held, void* workspace,
                               int64_t workspace_bytes, hipStream_t stream) {
    const int64_t need = vramc_kv_select_workspace(c, table_width, batch, count);
    if (need < 0) return (int)need;
    if (q_heads <= 0 || q_heads % c->kv_heads || first < 0 || last < 1 || (int64_t)first + last > count) return RANS_EARG;
    if (batch == 0) return 0;
    if (!bounds || (uintptr_t)bounds % 16 || !q || !lengths || !chosen || !held || (table_width && !table))
        return RANS_EARG;
    if (need && (!workspace || workspace_bytes < need)) return RANS_EWORKSPACE;
    if (need && (uintptr_t)workspace % 16) return RANS_EARG;
    const int lanes = lanes_of(c->head_dim), in_block = kWaves * kSets * 64 / lanes;
    const Select a{bounds, q, q_seq, q_head, q_heads / c->kv_heads, c->kv_heads, c->head_dim, lanes, c->pages,
                   __builtin_ctz(c->page_size), table, table_row, table_width, lengths, batch, count, first, last,
                   (table_width + in_block - 1) / in_block, static_cast<uint64_t*>(workspace), chosen, held};
    const int64_t rows = (int64_t)batch * c->kv_heads;
    if (need) {
        const dim3 grid((unsigned)(rows * a.chunks)), block(kThreads);
        if (c->dtype == RANS_X_F32) hipLaunchKernelGGL((score_kernel<float>), grid, block, 0, stream, a);
        else if (c->dtype == RANS_X_BF16) hipLaunchKernelGGL((score_kernel<__bf16>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((score_kernel<_Float16>), grid, block, 0, stream, a);
        if (const int rc = (int)hipGetLastError()) return rc;
    }
    hipLaunchKernelGGL(choose_kernel, dim3((unsigned)rows), dim3(kChoose), 0, stream, a);
    return (int)hipGetLastError();
}
