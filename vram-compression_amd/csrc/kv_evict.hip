// Eviction of a cache's tokens by accumulated weight.
//
// A kv head of a sequence ranks its tokens by a 32-bit key that sorts as the
// order of eviction does.  One workgroup reads the keys of up to 32768 tokens
// into LDS once, finds the budget-th largest by radix selection (11, 11 and 10
// bits, histograms in LDS too; the first digit is counted while the keys come
// in), and keeps every token above it and of those equal to it as many as there
// is room for, lowest index first.  A wave goes over neighbouring tokens, so
// that ranks within it are counts of ballot bits, and the order of indices
// costs one exchange between the waves.  Longer sequences go through in pieces
// of 32768 tokens, read again for every step.
//
// What moves is then two ordered lists of places, all different, and moving a
// copy of rows.  In place a kept token moves only if it lies beyond the budget:
// a decode step's eviction moves one token, not the cache.
//
// Selection is bound by the latency of its steps (reads, digits, lists) on one
// workgroup a head, moving by HBM: 8 heads of 4 sequences of 32768 tokens cut to
// 4096 take 23 us and then 134 MB, read and written, 30 us (4.4 TB/s); 2 heads of
// 64 sequences of 2049 cut to 2048 10.9 us in one launch, where two take 12.6.  One
// sequence of 131072 tokens, in pieces, cut to 16384 takes 151 us in all.
#include "kv_device.h"

namespace {

constexpr int kSelect = 1024;          // threads that select
constexpr int kWaves = kSelect / 64;
constexpr int kKeys = 32;              // keys of a lane
constexpr int kPiece = kSelect * kKeys;
constexpr int kBins = 2 * kSelect;     // of a digit of 11 bits
constexpr int kMove = 256;             // threads that move
constexpr int kRows = 16;              // tokens that a wave moves at once
// With at most this many moves a kv head (known from the table's width and the
// budget) the selecting workgroup makes them itself, a wave's worth each:
// a launch less.
constexpr int kMovesHere = kWaves * kRows;

struct Evict {
    vramc_kv_cache c;
    int page_shift;
    const int32_t* table;
    int64_t table_row;
    int bound;                   // tokens that a row of the table has room for
    const int32_t *lengths, *seen;
    int budget, recent;
    const int32_t* into;
    int64_t into_row;
    int32_t* new_lengths;
    int32_t *from, *to, *count;  // [batch * kv_heads][most] indices, and how many
    int most;
};

// The place of token j: slot of the cache for a kv head, -1 for none.
__device__ __forceinline__ int64_t place(const Evict& e, const int32_t* row, int h, int j) {
    const int page = row[j >> e.page_shift];
    if (page < 0 || page >= e.c.pages) return -1;
    return ((((int64_t)page * e.c.kv_heads + h) << e.page_shift) + (j & (e.c.page_size - 1)));
}

// The i-th index of a row that has a page; there are more than i.
__device__ __forceinline__ int nth_place(const Evict& e, const int32_t* row, int i) {
    for (int k = 0;; k++) {
        if ((uint32_t)row[k] >= (uint32_t)e.c.pages) continue;
        if (i < e.c.page_size) return (k << e.page_shift) + i;
        i -= e.c.page_size;
    }
}

// Sorts as the order in which tokens are kept: 1 for a token that is nowhere,
// the mass's bits made monotonic (NaN as -infinity), all ones for a recent one.
// 0 stands behind a sequence's last token and is never among the kept.
__device__ __forceinline__ uint32_t rank_of(float m, int position, bool there, int recent) {
    if (m != m) m = -__builtin_inff();
    const uint32_t bits = __float_as_uint(m + 0.f);  // -0 as 0
    const uint32_t sorted = bits >> 31 ? ~bits : bits | 0x80000000u;
    return !there ? 1 : position >= recent ? 0xffffffffu : sorted;
}

// What a wave's lanes wrote to or read from LDS before, for its other lanes that
// read or write there next.
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Copies the tokens of list entries first .. first + kRows - 1, below count, of
// a kv head, by one wave: 16 bytes a lane, two loads of keys and two of values
// before the first store (16 sequences of 16384 tokens in 4 bits cut to 2048: 37.4
// us, with four 39.5), the stores past the caches (4 sequences of 32768 in bf16 cut
// to 4096: 52.7 us against 57.1; the former 37.4 against 40.1).
__device__ __forceinline__ void move_rows(const Evict& e, int group, int first, int count, int64_t* from_at,
                          int64_t* to_at) {
    const int lane = threadIdx.x & 63, b = group / e.c.kv_heads, h = group % e.c.kv_heads;
    const int n = min(kRows, count - first);
    if (lane < kRows) {
        int64_t from = -1, to = -1;
        if (lane < n) {
            const int64_t i = (int64_t)group * e.most + first + lane;
            const int32_t* row = e.table + b * e.table_row;
            from = place(e, row, h, e.from[i]);
            to = place(e, e.into ? e.into + b * e.into_row : row, h, e.to[i]);
        }
        const bool moves = from >= 0 && to >= 0;
        from_at[lane] = moves ? from : -1;
        to_at[lane] = to;
        if (moves) {
            const float m = e.c.mass[from];
            const int p = e.c.position[from];
            e.c.mass[to] = m;
            e.c.position[to] = p;
        }
    }
    wave_order();
    const int wide = e.c.mx ? e.c.head_dim / 32 : e.c.head_dim * (e.c.dtype == RANS_X_F32 ? 4 : 2) / 16;
    auto* k = static_cast<vec<uint32_t, 4>*>(e.c.k);
    auto* v = static_cast<vec<uint32_t, 4>*>(e.c.v);
    constexpr int U = 2;
    for (int at = lane; at < n * wide; at += 64 * U) {
        vec<uint32_t, 4> x[U], y[U];
        int64_t to[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = at + 64 * u, r = i / wide;
            to[u] = -1;
            if (r < n && from_at[r] >= 0) {
                const int64_t from = from_at[r] * wide + (i - r * wide);
                to[u] = to_at[r] * wide + (i - r * wide);
                x[u] = k[from];
                y[u] = v[from];
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (to[u] >= 0) {
                __builtin_nontemporal_store(x[u], k + to[u]);
                __builtin_nontemporal_store(y[u], v + to[u]);
            }
    }
    if (e.c.mx) {
        const int scales = e.c.head_dim / kMxBlock;
        for (int i = lane; i < n * scales; i += 64) {
            const int r = i / scales;
            if (from_at[r] < 0) continue;
            const int64_t from = from_at[r] * scales + (i - r * scales);
            const int64_t to = to_at[r] * scales + (i - r * scales);
            const uint8_t x = e.c.k_scale[from], y = e.c.v_scale[from];
            e.c.k_scale[to] = x;
            e.c.v_scale[to] = y;
        }
    }
}

// The sum over a wave's lanes below this one, and over the workgroup's waves
// below this one; the workgroup's whole sum in *all.
__device__ __forceinline__ uint32_t before_of(uint32_t x, uint32_t* waves, uint32_t* all) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t sum = wave_scan((int)x);
    __syncthreads();
    if (lane == 63) waves[wave] = sum;
    __syncthreads();
    uint32_t below = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) {
        below += w < wave ? waves[w] : 0;
        total += waves[w];
    }
    *all = total;
    return below + sum - x;
}

// The n lowest bits of a word, and of those that are set in x.
__device__ __forceinline__ uint64_t low_bits(int n) {
    return n >= 64 ? ~0ull : n <= 0 ? 0 : (1ull << n) - 1;
}
__device__ __forceinline__ uint64_t lowest_set(uint64_t x, int n) {
    if (n <= 0) return 0;
    if (n >= (int)__popcll(x)) return x;
    int at = 0;  // of the n-th set bit, found by halves
#pragma unroll
    for (int half = 32; half; half /= 2) {
        const int in = __popcll(x >> at & low_bits(half));
        if (in < n) n -= in, at += half;
    }
    return x & low_bits(at + 1);
}

__global__ void __launch_bounds__(kSelect) select_kernel(Evict e, bool moves_here) {
    extern __shared__ __attribute__((aligned(16))) uint32_t piece_keys[];
    __shared__ int hist[kBins], found[3];
    __shared__ int absent, gaps;  // tokens, and places of the other pages, that have no page
    __shared__ uint32_t waves[kWaves];
    __shared__ int64_t rows[kWaves][2][kRows];
    const int b = blockIdx.x / e.c.kv_heads, h = blockIdx.x % e.c.kv_heads;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = min(max(e.lengths[b], 0), e.bound);
    const int32_t* row = e.table + b * e.table_row;
    const int32_t* other = e.into ? e.into + b * e.into_row : nullptr;
    const int recent = (int)max((int64_t)e.seen[b] - e.recent, (int64_t)INT32_MIN);
    const int keep = min(n, e.budget);
    if (h == 0 && threadIdx.x == 0) e.new_lengths[b] = keep;
    int32_t* from = e.from + (int64_t)blockIdx.x * e.most;
    int32_t* to = e.to + (int64_t)blockIdx.x * e.most;
    int count = 0;
    // Of the first `keep` places those without a page stay empty, and as many fewer
    // tokens are kept.  In place there are never fewer tokens than places, as those
    // below the budget lie in them; for other pages there may be.
    bool select = n > e.budget;
    // How many of the first `tokens` of a row have no page; the thread's first page
    // was read before.
    const auto without_page = [&](const int32_t* r, int tokens, int page, int* sum) {
        for (int k = threadIdx.x; k << e.page_shift < tokens; k += kSelect) {
            if (k >= kSelect) page = r[k];
            if ((uint32_t)page >= (uint32_t)e.c.pages)
                atomicAdd(sum, min(e.c.page_size, tokens - (k << e.page_shift)));
        }
    };
    int to_page = 0;
    if (select || e.into) {
        hist[threadIdx.x] = hist[threadIdx.x + kSelect] = 0;
        if (threadIdx.x == 0) absent = gaps = 0;
        const bool mine = (int)threadIdx.x << e.page_shift < keep;
        if (e.into && mine) to_page = other[threadIdx.x];
        __syncthreads();
        if (!select) {  // everything is kept, in its order, where every page is there
            const int page = mine ? row[threadIdx.x] : 0;
            without_page(other, keep, to_page, &gaps);
            without_page(row, n, page, &absent);
            __syncthreads();
            select = absent | gaps;
            __syncthreads();
            if (threadIdx.x == 0) absent = gaps = 0;  // counted again with the keys
            __syncthreads();
            if (!select) {
                count = n;
                for (int j = threadIdx.x; j < n; j += kSelect) from[j] = to[j] = j;
            }
        }
    }
    if (select) {
        const int pieces = (n + kPiece - 1) / kPiece;
        // keys of a lane, in fours
        const int each = pieces > 1 ? kKeys : (n + 4 * kSelect - 1) / (4 * kSelect) * 4;
        int first, limit;  // the wave's tokens in the piece at hand, and its keys
        uint32_t* keys = piece_keys + wave * 64 * each + lane;
        const auto load = [&](int piece, bool count) {
            first = piece * kPiece + wave * 64 * each;
            limit = min(n, first + 64 * each);
            // the wave's pages: at most 2048 tokens, 16 or more to a page
            const int page0 = first >> e.page_shift, last = (max(limit, 1) - 1) >> e.page_shift;
            int page[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                page[u] = page0 + 64 * u + lane <= last ? row[page0 + 64 * u + lane] : -1;
                if ((uint32_t)page[u] >= (uint32_t)e.c.pages) page[u] = -1;
            }
            // four neighbouring tokens a lane, 256 a wave, all loads before the first use
            vec<uint32_t, 4>* to = reinterpret_cast<vec<uint32_t, 4>*>(piece_keys + wave * 64 * each) + lane;
            vec<float, 4> m[kKeys / 4];
            vec<int, 4> p[kKeys / 4];
            uint32_t there = 0;
#pragma unroll
            for (int u = 0; u < kKeys / 4; u++)
                if (4 * u < each && first + 256 * u < limit) {
                    const int j = min(first + 256 * u + 4 * lane, limit - 1) & ~3;
                    const int k = (j >> e.page_shift) - page0;
                    const int x = __shfl(page[0], k & 63), y = __shfl(page[1], k & 63);
                    const int in = k < 64 ? x : y;
                    there |= (uint32_t)(in >= 0) << u;
                    const int64_t at = ((((int64_t)max(in, 0) * e.c.kv_heads + h) << e.page_shift) +
                                        (j & (e.c.page_size - 1)));
                    m[u] = *reinterpret_cast<const vec<float, 4>*>(e.c.mass + at);
                    p[u] = *reinterpret_cast<const vec<int, 4>*>(e.c.position + at);
                }
            if (count) {
                const int stop = e.into ? limit : min(limit, keep);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int lost = min(e.c.page_size, stop - ((page0 + 64 * u + lane) << e.page_shift));
                    if (page[u] < 0 && lost > 0) atomicAdd(&absent, lost);
                }
            }
            wave_order();  // other lanes have read the last piece's keys
#pragma unroll
            for (int u = 0; u < kKeys / 4; u++)
                if (4 * u < each) {
                    vec<uint32_t, 4> r = {};
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (first + 256 * u + 4 * lane + i < limit) {
                            r[i] = rank_of(m[u][i], p[u][i], there >> u & 1, recent);
                            if (count) atomicAdd(&hist[r[i] >> 21], 1);
                        }
                    to[64 * u] = r;
                }
            wave_order();
        };
        const auto over_keys = [&](auto f) {  // f(i, key): the wave's tokens 64 * i..
            for (int i = 0; i < each; i += 4) {
                uint32_t r[4];
#pragma unroll
                for (int u = 0; u < 4; u++) r[u] = keys[64 * (i + u)];
#pragma unroll
                for (int u = 0; u < 4; u++) f(i + u, r[u]);
            }
        };
        uint32_t above = 0;  // the digits found so far
        int room = 0;        // tokens to keep of those that share them
        int in_bin = 0;      // and how many do
        if (pieces == 1) load(0, true);  // the first digit is counted on the way
        if (e.into) without_page(other, keep, to_page, &gaps);
        for (int shift = 21, bits = 11;; shift = shift == 21 ? 10 : 0) {
            for (int piece = 0; piece < pieces; piece++) {
                if (pieces > 1) load(piece, shift == 21);
                if (shift < 21)
                    over_keys([&](int, uint32_t r) {
                        if (r && (r ^ above) >> (shift + bits) == 0)
                            atomicAdd(&hist[r >> shift & ((1 << bits) - 1)], 1);
                    });
            }
            __syncthreads();
            if (shift == 21) {
                // tokens that there are, and places for them
                room = e.into ? min(n - absent, keep - gaps) : keep - absent;
                if (e.into && h == 0 && threadIdx.x == 0 && room < keep - gaps)
                    e.new_lengths[b] = room ? nth_place(e, other, room - 1) + 1 : 0;
                if (room == 0) break;
            }
            // the bin that holds the room-th largest: a sum from the top over
            // the threads, two bins each
            const int low = hist[2 * threadIdx.x], high = hist[2 * threadIdx.x + 1];
            const int sum = wave_scan(low + high);
            if (lane == 63) waves[wave] = sum;
            __syncthreads();
            hist[2 * threadIdx.x] = hist[2 * threadIdx.x + 1] = 0;
            int over = -sum;  // in the bins above these two
#pragma unroll
            for (int w = 0; w < kWaves; w++) over += w >= wave ? waves[w] : 0;
            if (over < room && room <= over + low + high) {
                const bool upper = room <= over + high;
                found[0] = 2 * threadIdx.x + upper;
                found[1] = room - over - (upper ? 0 : high);
                found[2] = upper ? high : low;
            }
            __syncthreads();
            above |= (uint32_t)found[0] << shift;
            room = found[1];
            in_bin = found[2];
            if (room == in_bin || shift == 0) break;  // all that share these digits are kept
            bits = shift == 21 ? 11 : 10;
        }
        // Kept: what exceeds `above`, which has the digits found and zeros behind
        // them, and `room` of those that share its digits.  If the search ended
        // early those are all that there are, else they are equal to it.
        const bool all = room == in_bin;
        above = max(above, 1u);  // not what stands behind the last token
        const bool holes = absent && !e.into;
        // Lane i of a wave decides about its i-th 64 tokens, all bits at once.
        uint32_t ties = 0, lists[2] = {0, 0};  // of the pieces so far
        for (int piece = 0; room && piece < pieces; piece++) {
            if (pieces > 1) load(piece, false);
            uint64_t more = 0, same = 0;
            over_keys([&](int i, uint32_t r) {
                const uint64_t x = __ballot(r > above), y = __ballot(r == above);
                if (lane == i) more = x, same = y;
            });
            uint32_t sum;
            if (!all) {
                const uint32_t before = ties + before_of(__popcll(same), waves, &sum);
                ties += sum;
                same = lowest_set(same, room - (int)before);
            }
            const int start = first + 64 * lane;  // of the lane's 64 tokens
            const uint64_t kept = more | same, low = low_bits(e.budget - start);
            uint64_t there = low_bits(limit - start);
            if (holes)
                over_keys([&](int i, uint32_t r) {
                    const uint64_t x = __ballot(r > 1);
                    if (lane == i) there &= x;
                });
            const uint64_t listed[2] = {e.into ? kept : there & low & ~kept,
                                        e.into ? 0 : kept & ~low};
            // at most 32768 of each in a piece: both sums in one word
            const uint32_t before = before_of(__popcll(listed[0]) | __popcll(listed[1]) << 16, waves, &sum);
            const uint32_t at[2] = {lists[0] + (before & 0xffff), lists[1] + (before >> 16)};
            lists[0] += sum & 0xffff;
            lists[1] += sum >> 16;
            // and writes its own down, each half of the wave 32 bits of the 64
#pragma unroll
            for (int k = 0; k < 2; k++) {
                if (k && e.into) break;
                const uint32_t x = __shfl((int)(uint32_t)listed[k], lane & 31);
                const uint32_t y = __shfl((int)(uint32_t)(listed[k] >> 32), lane & 31);
                uint32_t left = lane < 32 ? x : y;
                int i = __shfl((int)at[k], lane & 31) + (lane < 32 ? 0 : __popc(x));
                for (int j = first + 64 * (lane & 31) + (lane & 32); left; left &= left - 1, i++) {
                    const int token = j + __builtin_ctz(left);
                    if (e.into) {
                        to[i] = i;
                        from[i] = token;
                    } else {
                        (k ? from : to)[i] = token;
                    }
                }
            }
        }
        count = lists[0];
        if (gaps) {  // of the other pages: to the places that there are
            __syncthreads();
            for (int i = threadIdx.x; i < count; i += kSelect) to[i] = nth_place(e, other, i);
        }
    }
    if (!moves_here) {
        if (threadIdx.x == 0) e.count[blockIdx.x] = count;
        return;
    }
    __syncthreads();  // the lists are this workgroup's own
    if (wave * kRows < count) move_rows(e, blockIdx.x, wave * kRows, count, rows[wave][0], rows[wave][1]);
}

__global__ void __launch_bounds__(kMove) move_kernel(Evict e) {
    __shared__ int64_t rows[kMove / 64][2][kRows];
    const int wave = threadIdx.x >> 6, group = blockIdx.y;
    const int first = (blockIdx.x * (kMove / 64) + wave) * kRows, count = e.count[group];
    if (first < count) move_rows(e, group, first, count, rows[wave][0], rows[wave][1]);
}

// Lets the selecting workgroup have more LDS than 64 KB on the current device.
int allow_lds() {
    return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(select_kernel),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, kPiece * 4);
}

// Tokens of a kv head that one call can move.
int64_t most_moves(const vramc_kv_cache& c, int table_width, int budget, bool into) {
    const int64_t bound = (int64_t)table_width * c.page_size;
    if (into) return budget < bound ? budget : bound;
    const int64_t over = bound > budget ? bound - budget : 0;
    return budget < over ? budget : over;
}

// Whether n integers at a share memory with rows of `wide` at b, `step` apart.
bool overlap(const int32_t* a, int64_t n, const int32_t* b, int64_t step, int64_t wide, int64_t rows) {
    const auto meets = [&](int64_t from, int64_t to) {  // integers of b
        return (uintptr_t)a < (uintptr_t)(b + to) && (uintptr_t)(b + from) < (uintptr_t)(a + n);
    };
    const int64_t last = step * (rows - 1);
    bool any = wide > 0 && meets(last < 0 ? last : 0, (last > 0 ? last : 0) + wide);
    if (any && rows > 1) {  // or only with what lies between the rows
        any = false;
        for (int64_t r = 0; r < rows && !any; r++) any = meets(r * step, r * step + wide);
    }
    return any;
}

}  // namespace

extern "C" int64_t vramc_kv_evict_workspace(const vramc_kv_cache* c, int table_width, int batch,
                                            int budget, int into) {
    if (const int rc = check_cache(c)) return rc;
    if (!c->mass || table_width < 0 || batch < 0 || budget <= 0 ||
        (int64_t)table_width * c->page_size > kMaxTokens || (int64_t)batch * c->kv_heads > 65535)
        return RANS_EARG;
    return (int64_t)batch * c->kv_heads * (4 + 8 * most_moves(*c, table_width, budget, into));
}

extern "C" int vramc_kv_evict(const vramc_kv_cache* c, const int32_t* table, int64_t table_row,
                              int table_width, const int32_t* lengths, const int32_t* seen,
                              int batch, int budget, int recent, const int32_t* into,
                              int64_t into_row, int into_width, int32_t* new_lengths,
                              void* workspace, int64_t workspace_bytes, hipStream_t stream) {
    const int64_t need = vramc_kv_evict_workspace(c, table_width, batch, budget, into != nullptr);
    if (need < 0) return (int)need;
    if (batch == 0) return 0;
    if (!lengths || !seen || !new_lengths || (table_width && !table) || recent < 0) return RANS_EARG;
    const int64_t most = most_moves(*c, table_width, budget, into != nullptr);
    if (into && (int64_t)into_width * c->page_size < most) return RANS_EARG;
    if (!workspace || workspace_bytes < need) return RANS_EWORKSPACE;
    // Workgroups read all of these while others write the new lengths.
    if ((uintptr_t)workspace % 16 || overlap(new_lengths, batch, lengths, 0, batch, 1) ||
        overlap(new_lengths, batch, seen, 0, batch, 1) ||
        overlap(new_lengths, batch, table, table_row, table_width, batch) ||
        (into && overlap(new_lengths, batch, into, into_row, into_width, batch)))
        return RANS_EARG;
    const int64_t heads = (int64_t)batch * c->kv_heads;
    auto* count = static_cast<int32_t*>(workspace);
    Evict e{*c, __builtin_ctz(c->page_size), table, table_row, table_width * c->page_size, lengths,
            seen, budget, recent, into, into_row, new_lengths, count + heads,
            count + heads + heads * most, count, (int)most};
    const bool here = most <= kMovesHere;
    const int64_t keys = e.bound < kPiece ? e.bound : kPiece;
    const size_t lds = (size_t)((keys + 4 * kSelect - 1) / (4 * kSelect) * (4 * kSelect) * 4);
    if (lds > 32768)  // with what the kernel has besides, up to 64 KB need no leave
        if (const int rc = allow_lds()) return rc;
    hipLaunchKernelGGL(select_kernel, dim3((unsigned)heads), dim3(kSelect), lds, stream, e, here);
    if (const int rc = (int)hipGetLastError()) return rc;
    if (here) return 0;
    const int rows = kMove / 64 * kRows;
    hipLaunchKernelGGL(move_kernel, dim3((unsigned)((most + rows - 1) / rows), (unsigned)heads),
                       dim3(kMove), 0, stream, e);
    return (int)hipGetLastError();
}
