// Pages for new tokens, and back: a step's block table and slots from lengths.
//
// A call is latency: a few reads of each sequence, two sums over all of them, and
// 16 bytes for each token.  extend is one launch: every workgroup makes both sums
// over all sequences by itself (4096 at most, 16 to a thread), which takes less
// than a second launch, and then takes some of the rows, whose sequences it finds in
// LDS.  What is written (entries behind a sequence's pages, other tensors) nobody
// reads, but for the stack's count, which the workgroup that ends last sets.  One token
// each of 64 sequences 4.0 us in a trace, and 2.8 + 2.8 to take pages back from their 512
// entries each; in a graph 8.9 together.
#include "kv_device.h"

#include "../../include/vramc_pages.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
// Workgroups of extend, which takes more rows in turns: each makes the sums again and
// ends with a count in one place of memory (16 sequences of up to 8000 new tokens 7.5 us,
// by 1024 workgroups 8.6).
constexpr int kMaxBlocks = 256;
constexpr int kMaxBatch = 4096;
constexpr int kTurns = 4;                  // entries of a thread at once

struct Extend {
    vramc_pages p;
    int page_shift;
    int32_t* table;
    int64_t table_row;
    int width;
    const int32_t *lengths, *fresh, *seen;
    int batch, tokens;
    int64_t* slots;
    int32_t *positions, *filled, *starts, *new_lengths;
};

// The sum over the threads before this one.
__device__ __forceinline__ int64_t before_of(int64_t x, int64_t* waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t sum = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int64_t y = __shfl_up(sum, d);
        if (lane >= d) sum += y;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = sum;
    __syncthreads();
    int64_t below = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) below += w < wave ? waves[w] : 0;
    return below + sum - x;
}

__global__ void __launch_bounds__(kThreads) extend_kernel(Extend e) {
    extern __shared__ int32_t shared[];
    // first new tokens, then where a sequence's rows end; pages that it holds; pages
    // taken before its own, -1 without room
    int32_t *ends = shared, *held = shared + e.batch, *from = shared + 2 * e.batch;
    __shared__ int64_t waves[kWaves];
    __shared__ int taken;
    const int shift = e.page_shift, room = e.width << shift, each = (e.batch + kThreads - 1) / kThreads;
    const int b0 = min((int)threadIdx.x * each, e.batch), b1 = min(b0 + each, e.batch);
    const int have = min(max(*e.p.count, 0), e.p.pages);
    const auto pages_of = [&](int64_t n) { return (int)((n + (1 << shift) - 1) >> shift); };
    // pages that a sequence of n tokens wants for m more, whose rows end at `end`
    const auto want = [&](int n, int m, int64_t end, bool* fits) {
        *fits = (int64_t)n + m <= room && end <= e.tokens;
        return *fits ? pages_of(n + m) - pages_of(n) : 0;
    };
    if (threadIdx.x == 0) taken = 0;
    int64_t sum = 0, pages = 0;
    bool fits;
    for (int b = b0; b < b1; b++) {
        const int m = (int)min((uint32_t)max(e.fresh[b], 0), (uint32_t)e.tokens + 1);
        held[b] = min(max(e.lengths[b], 0), room);
        ends[b] = m;
        sum += m;
    }
    const int64_t start = before_of(sum, waves);
    sum = start;
    for (int b = b0; b < b1; b++) pages += want(held[b], ends[b], sum += ends[b], &fits);
    pages = before_of(pages, waves);
    sum = start;
    for (int b = b0; b < b1; b++) {
        const int n = held[b], m = ends[b];
        if (blockIdx.x == 0) e.starts[b] = (int)min(sum, (int64_t)e.tokens);
        sum += m;
        const int need = want(n, m, sum, &fits);
        const bool served = fits && (need == 0 || pages + need <= have);
        ends[b] = (int)min(sum, (int64_t)e.tokens);
        from[b] = !served ? -1 : need ? (int)pages : 0;
        pages += need;
        if (served && need) atomicMax(&taken, (int)pages);  // those that are served come first
        if (blockIdx.x == 0) e.new_lengths[b] = n + (served ? m : 0);
    }
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) e.starts[e.batch] = e.batch ? ends[e.batch - 1] : 0;
#pragma unroll 1
    for (int64_t row = (int64_t)blockIdx.x * kThreads + threadIdx.x; row < e.tokens; row += (int64_t)gridDim.x * kThreads) {
        const int t = (int)row;
        int b = 0;  // the first sequence that ends behind t
#pragma unroll 1
        for (int n = e.batch; n > 0;) {
            const int half = n / 2;
            const bool behind = ends[b + half] <= t;
            b = behind ? b + half + 1 : b;
            n = behind ? n - half - 1 : half;
        }
        int page = -1, place = 0, position = 0;
        if (b < e.batch) {
            const int in = t - (b ? ends[b - 1] : 0), n = held[b];
            if (from[b] >= 0) {
                const int index = n + in, old = pages_of(n), k = index >> shift;
                place = index & ((1 << shift) - 1);
                int32_t* entry = e.table + b * e.table_row + k;
                page = *(k < old ? entry : e.p.free + (have - 1 - (from[b] + k - old)));
                if ((uint32_t)page >= (uint32_t)e.p.pages) page = -1;
                if (k >= old && place == 0) *entry = page;
            }
            position = (int)((uint32_t)(e.seen ? e.seen[b] : n) + (uint32_t)in);
        }
        e.slots[t] = page < 0 ? -1 : ((int64_t)page << shift) + place;
        e.positions[t] = position;
        e.filled[t] = place == (1 << shift) - 1 ? page : -1;
    }
    __syncthreads();
    if (threadIdx.x) return;
    if (gridDim.x > 1) {  // the workgroups have all read the count when the last of them is here
        if (__hip_atomic_fetch_add((uint32_t*)e.p.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != gridDim.x - 1)
            return;
        *e.p.ticket = 0;
    }
    *e.p.count = have - taken;
}

struct Release {
    vramc_pages p;
    int page_shift;
    int32_t* table;
    int64_t table_row;
    int width;
    const int32_t* lengths;
    int batch;
    int32_t *counts, *base;  // pages that each row gives back, and the stack's count before

    // entries that a row keeps
    __device__ __forceinline__ int kept(int b) const {
        const int n = min(max(lengths[b], 0), width << page_shift);
        return (n + (1 << page_shift) - 1) >> page_shift;
    }
    __device__ __forceinline__ bool is_page(int x) const { return (uint32_t)x < (uint32_t)p.pages; }
};

// The sum over the workgroup.
__device__ __forceinline__ int sum_of(int x, int* waves) {
#pragma unroll
    for (int d = 32; d; d /= 2) x += __shfl_xor(x, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = x;
    __syncthreads();
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kWaves; w++) sum += waves[w];
    return sum;
}

// Small tables by one workgroup: pieces of 256 entries of a row, up to kPieces to each
// of its waves, four neighbouring entries to a lane, read once, counted, and then put
// behind what the waves before have.  With extend, of one token each: a row of 512
// entries 5.7 us, and 7.2 where two launches give pages back, 16 rows 7.8 and 9.3, 64
// rows of 256 11.4 and 10.7, where a launch less is worth more to a host that is waited
// for (2.7 us); 64 of 512, with twice the pieces, 14.5 and 11.0.
constexpr int kAll = 1024, kAllWaves = kAll / 64, kPieces = 4;

__global__ void __launch_bounds__(kAll) release_kernel(Release r) {
    __shared__ int waves[kAllWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per_row = (r.width + 255) / 256, all = per_row * r.batch, each = (all + kAllWaves - 1) / kAllWaves;
    const int first = min(wave * each, all - 1), mine = min(each, all - wave * each);
    const int b0 = first / per_row, c0 = first - b0 * per_row;
    const int have = min(max(*r.p.count, 0), r.p.pages);
    using Four = vec<int, 4>;
    Four x[kPieces];
    int kept[kPieces];
    const auto over = [&](auto f) {  // f(u, row, first of the lane's entries)
        int b = b0, c = c0;
#pragma unroll
        for (int u = 0; u < kPieces; u++) {
            if (u < mine) f(u, b, 256 * c + 4 * lane);
            if (++c == per_row) c = 0, b++;
        }
    };
    over([&](int u, int b, int i) {
        x[u] = *reinterpret_cast<const Four*>(r.table + b * r.table_row + min(i, r.width - 4));
        kept[u] = r.kept(b);
    });
    int n = 0;
    over([&](int u, int, int i) {
#pragma unroll
        for (int e = 0; e < 4; e++) n += __popcll(__ballot((i < r.width) & (i + e >= kept[u]) & r.is_page(x[u][e])));
    });
    if (lane == 0) waves[wave] = n;
    __syncthreads();
    int at = have, total = have;
#pragma unroll
    for (int w = 0; w < kAllWaves; w++) {
        at += w < wave ? waves[w] : 0;
        total += waves[w];
    }
    over([&](int u, int b, int i) {
        Four y = x[u];
        uint32_t to = at;
        bool goes[4], changes = false;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool behind = (i < r.width) & (i + e >= kept[u]);
            goes[e] = behind & r.is_page(x[u][e]);
            changes |= behind & (x[u][e] != -1);
            y[e] = behind ? -1 : x[u][e];
            const uint64_t mask = __ballot(goes[e]);
            to = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, to));
            at += __popcll(mask);
        }
        if (!__any(changes)) return;
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (goes[e]) {
                if (to < (uint32_t)r.p.pages) r.p.free[to] = x[u][e];
                to++;
            }
        if (changes) *reinterpret_cast<Four*>(r.table + b * r.table_row + i) = y;
    });
    if (threadIdx.x == 0) *r.p.count = min(total, r.p.pages);
}

// Larger tables, a workgroup to a row: how many pages it gives back, and then, in a
// second launch, those behind what the rows before it do.
__global__ void __launch_bounds__(kThreads) release_count_kernel(Release r) {
    __shared__ int waves[kWaves];
    const int b = blockIdx.x;
    int32_t* row = r.table + b * r.table_row;
    int n = 0;
    for (int i = r.kept(b) + threadIdx.x; i < r.width; i += kThreads) {
        const int x = row[i];
        n += r.is_page(x);
        if (!r.is_page(x) && x != -1) row[i] = -1;
    }
    n = sum_of(n, waves);
    if (threadIdx.x) return;
    r.counts[b] = n;
    if (b == 0) *r.base = min(max(*r.p.count, 0), r.p.pages);
}

__global__ void __launch_bounds__(kThreads) release_rows_kernel(Release r) {
    __shared__ int waves[kWaves], found[kTurns][kWaves];
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mine = r.counts[b];
    if (mine == 0 && b != r.batch - 1) return;
    int before = 0;
    for (int i = threadIdx.x; i < b; i += kThreads) before += r.counts[i];
    int at = *r.base + sum_of(before, waves);
    if (b == r.batch - 1 && threadIdx.x == 0) *r.p.count = min(at + mine, r.p.pages);
    if (mine == 0) return;
    int32_t* row = r.table + b * r.table_row;
    for (int first = r.kept(b); first < r.width; first += kTurns * kThreads) {
        int x[kTurns];
        uint64_t back[kTurns];
#pragma unroll
        for (int u = 0; u < kTurns; u++) {
            const int i = first + u * kThreads + threadIdx.x;
            x[u] = i < r.width ? row[i] : -1;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kTurns; u++) {
            back[u] = __ballot(r.is_page(x[u]));
            if (lane == 0) found[u][wave] = __popcll(back[u]);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kTurns; u++) {
            int to = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(back[u] >> 32),
                                                    __builtin_amdgcn_mbcnt_lo((uint32_t)back[u], 0));
#pragma unroll
            for (int w = 0; w < kWaves; w++) {
                to += w < wave ? found[u][w] : 0;
                at += found[u][w];
            }
            if (r.is_page(x[u])) {
                if (to < r.p.pages) r.p.free[to] = x[u];
                row[first + u * kThreads + threadIdx.x] = -1;
            }
        }
    }
}

int check_pool(const vramc_pages* p) {
    if (!p || !p->free || !p->count || !p->ticket || p->pages <= 0) return RANS_EARG;
    switch (p->page_size) {
        case 16: case 32: case 64: case 128: case 256: return 0;
        default: return RANS_EUNSUPPORTED;
    }
}
int check_table(const vramc_pages* p, int64_t table_row, int table_width, int batch) {
    if (const int rc = check_pool(p)) return rc;
    if (table_width < 0 || batch < 0 || batch > kMaxBatch ||
        (int64_t)table_width * p->page_size > kMaxTokens || (batch > 1 && table_row < table_width))
        return RANS_EARG;
    return 0;
}

// Whether one workgroup takes the table.
bool one_launch(const int32_t* table, int64_t table_row, int table_width, int batch) {
    return ((uintptr_t)table % 16 | table_row % 4 | table_width % 4) == 0 &&
           (int64_t)((table_width + 255) / 256) * batch <= kAllWaves * kPieces;
}

// A pool's tensors.
struct PoolSpans {
    Span of[3];
};
PoolSpans spans_of(const vramc_pages& p) {
    return {{{p.free, (int64_t)p.pages * 4}, {p.count, 4}, {p.ticket, 4}}};
}

// Whether some of these share memory with one another.
template <size_t N>
bool overlap(const Span (&a)[N]) {
    for (size_t i = 0; i < N; i++)
        for (size_t j = 0; j < i; j++)
            if (overlap(a[i], a[j])) return true;
    return false;
}

}  // namespace

extern "C" int vramc_pages_extend(const vramc_pages* p, int32_t* table, int64_t table_row,
                                  int table_width, const int32_t* lengths, const int32_t* fresh,
                                  const int32_t* seen, int batch, int64_t tokens, int64_t* slots,
                                  int32_t* positions, int32_t* filled, int32_t* starts,
                                  int32_t* new_lengths, hipStream_t stream) {
    if (const int rc = check_table(p, table_row, table_width, batch)) return rc;
    if (tokens < 0 || tokens > INT32_MAX - 1 || !starts) return RANS_EARG;
    if (batch && (!lengths || !fresh || !new_lengths || (table_width && !table))) return RANS_EARG;
    if (tokens && (!slots || !positions || !filled)) return RANS_EARG;
    const Span out[] = {{slots, tokens * 8}, {positions, tokens * 4}, {filled, tokens * 4},
                        {starts, 4 * ((int64_t)batch + 1)}, {new_lengths, 4 * (int64_t)batch},
                        span_of(table, table_row, 0, batch, 1, table_width, 4)};
    const Span read[] = {{lengths, 4 * (int64_t)batch}, {fresh, 4 * (int64_t)batch}, {seen, 4 * (int64_t)batch}};
    const auto pool = spans_of(*p);
    if (overlap(out) || overlap(out, read) || overlap(out, pool.of) || overlap(pool.of) || overlap(pool.of, read))
        return RANS_EARG;
    const Extend e{*p, __builtin_ctz(p->page_size), table, table_row, table_width, lengths, fresh, seen, batch,
                   (int)tokens, slots, positions, filled, starts, new_lengths};
    const int64_t blocks = (tokens + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(extend_kernel, dim3(blocks == 0 ? 1 : blocks < kMaxBlocks ? (unsigned)blocks : kMaxBlocks), dim3(kThreads), (size_t)batch * 12, stream, e);
    return (int)hipGetLastError();
}

extern "C" int64_t vramc_pages_release_workspace(const vramc_pages* p, int table_width, int batch) {
    if (const int rc = check_table(p, table_width, table_width, batch)) return rc;
    return 4 * ((int64_t)batch + 1);
}

extern "C" int vramc_pages_release(const vramc_pages* p, int32_t* table, int64_t table_row,
                                   int table_width, const int32_t* lengths, int batch, void* workspace,
                                   int64_t workspace_bytes, hipStream_t stream) {
    if (const int rc = check_table(p, table_row, table_width, batch)) return rc;
    if (batch == 0 || table_width == 0) return 0;
    if (!table || !lengths) return RANS_EARG;
    if (!workspace || workspace_bytes < vramc_pages_release_workspace(p, table_width, batch)) return RANS_EWORKSPACE;
    if ((uintptr_t)workspace % 16) return RANS_EARG;
    const Span out[] = {span_of(table, table_row, 0, batch, 1, table_width, 4), {workspace, 4 * ((int64_t)batch + 1)}};
    const Span read[] = {{lengths, 4 * (int64_t)batch}};
    const auto pool = spans_of(*p);
    if (overlap(out) || overlap(out, read) || overlap(out, pool.of) || overlap(pool.of) || overlap(pool.of, read))
        return RANS_EARG;
    auto* counts = static_cast<int32_t*>(workspace);
    const Release r{*p, __builtin_ctz(p->page_size), table, table_row, table_width, lengths, batch, counts,
                    counts + batch};
    if (one_launch(table, table_row, table_width, batch)) {
        hipLaunchKernelGGL(release_kernel, dim3(1), dim3(kAll), 0, stream, r);
        return (int)hipGetLastError();
    }
    hipLaunchKernelGGL(release_count_kernel, dim3((unsigned)batch), dim3(kThreads), 0, stream, r);
    if (const int rc = (int)hipGetLastError()) return rc;
    hipLaunchKernelGGL(release_rows_kernel, dim3((unsigned)batch), dim3(kThreads), 0, stream, r);
    return (int)hipGetLastError();
}
