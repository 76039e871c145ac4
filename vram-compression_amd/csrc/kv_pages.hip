// Pages for new tokens, and back: a step's block table and slots from lengths.
//
// A call is latency: a few reads of each sequence, two sums over all of them, and
// 16 bytes for each token.  extend is one launch: every workgroup makes both sums
// over all sequences by itself (4096 at most, 16 to a thread), which takes less
// than a second launch, and then takes 1024 of the rows, whose sequences it finds in
// LDS.  What is written (entries behind a sequence's pages, other tensors) nobody
// reads, but for the stack's count, which the workgroup that ends last sets.
#include "kv_device.h"

#include "../../include/vramc_pages.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kRows = 4;                    // rows of a thread
constexpr int kMaxBatch = 4096;

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
    int32_t *ends = shared, *from = shared + e.batch;  // from: pages before a sequence's, -1 without room
    __shared__ int64_t waves[kWaves];
    __shared__ int taken;
    const int shift = e.page_shift, room = e.width << shift, each = (e.batch + kThreads - 1) / kThreads;
    const int b0 = min((int)threadIdx.x * each, e.batch), b1 = min(b0 + each, e.batch);
    const int have = min(max(*e.p.count, 0), e.p.pages);
    const auto length_of = [&](int b) { return min(max(e.lengths[b], 0), room); };
    const auto fresh_of = [&](int b) { return (int64_t)min((uint32_t)max(e.fresh[b], 0), (uint32_t)e.tokens + 1); };
    const auto pages_of = [&](int64_t n) { return (int)((n + (1 << shift) - 1) >> shift); };
    // pages that a sequence wants whose rows end at `end`
    const auto want = [&](int b, int64_t end, bool* fits) {
        const int64_t n = length_of(b), all = n + fresh_of(b);
        *fits = all <= room && end <= e.tokens;
        return *fits ? pages_of(all) - pages_of(n) : 0;
    };
    if (threadIdx.x == 0) taken = 0;
    int64_t sum = 0, pages = 0;
    bool fits;
    for (int b = b0; b < b1; b++) sum += fresh_of(b);
    const int64_t start = before_of(sum, waves);
    sum = start;
    for (int b = b0; b < b1; b++) pages += want(b, sum += fresh_of(b), &fits);
    pages = before_of(pages, waves);
    sum = start;
    for (int b = b0; b < b1; b++) {
        if (blockIdx.x == 0) e.starts[b] = (int)min(sum, (int64_t)e.tokens);
        sum += fresh_of(b);
        const int need = want(b, sum, &fits);
        const bool served = fits && (need == 0 || pages + need <= have);
        ends[b] = (int)min(sum, (int64_t)e.tokens);
        from[b] = !served ? -1 : need ? (int)pages : 0;
        pages += need;
        if (served && need) atomicMax(&taken, (int)pages);  // those that are served come first
        if (blockIdx.x == 0) e.new_lengths[b] = length_of(b) + (served ? (int)fresh_of(b) : 0);
    }
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) e.starts[e.batch] = e.batch ? ends[e.batch - 1] : 0;
#pragma unroll
    for (int i = 0; i < kRows; i++) {
        const int64_t row = ((int64_t)blockIdx.x * kRows + i) * kThreads + threadIdx.x;
        if (row >= e.tokens) break;
        const int t = (int)row;
        int b = 0;  // the first sequence that ends behind t
        for (int n = e.batch; n > 0;) {
            const int half = n / 2;
            const bool behind = ends[b + half] <= t;
            b = behind ? b + half + 1 : b;
            n = behind ? n - half - 1 : half;
        }
        int64_t slot = -1;
        int position = 0, full = -1;
        if (b < e.batch) {
            const int in = t - (b ? ends[b - 1] : 0), n = length_of(b);
            position = (int)((uint32_t)(e.seen ? e.seen[b] : n) + (uint32_t)in);
            if (from[b] >= 0) {
                const int index = n + in, old = pages_of(n), k = index >> shift, place = index & ((1 << shift) - 1);
                int32_t* entry = e.table + b * e.table_row + k;
                int page = k < old ? *entry : e.p.free[have - 1 - (from[b] + k - old)];
                if ((uint32_t)page >= (uint32_t)e.p.pages) page = -1;
                if (k >= old && place == 0) *entry = page;
                if (page >= 0) {
                    slot = ((int64_t)page << shift) + place;
                    if (place == (1 << shift) - 1) full = page;
                }
            }
        }
        e.slots[t] = slot;
        e.positions[t] = position;
        e.filled[t] = full;
    }
    __syncthreads();
    if (threadIdx.x) return;
    if (gridDim.x > 1) {  // the workgroups have all read the count when the last of them is here
        __threadfence();
        if (atomicAdd((uint32_t*)e.p.ticket, 1u) != gridDim.x - 1) return;
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
    int32_t *counts, *base;  // two launches: pages that each row gives back, and the stack's count before

    // entries that a row keeps
    __device__ __forceinline__ int kept(int b) const {
        const int n = min(max(lengths[b], 0), width << page_shift);
        return (n + (1 << page_shift) - 1) >> page_shift;
    }
    __device__ __forceinline__ bool is_page(int x) const { return (uint32_t)x < (uint32_t)p.pages; }
};

// Pieces of 64 entries of a row, kPieces to each of sixteen waves, in registers
// between their count and their place on the stack.
constexpr int kAll = 1024, kAllWaves = kAll / 64, kPieces = 32;

__global__ void __launch_bounds__(kAll) release_kernel(Release r) {
    __shared__ int waves[kAllWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per_row = (r.width + 63) / 64, all = per_row * r.batch, each = (all + kAllWaves - 1) / kAllWaves;
    const int have = min(max(*r.p.count, 0), r.p.pages);
    int x[kPieces], n = 0;
    const auto place = [&](int u, int* b, int* i) {
        const int s = wave * each + u;
        *b = min(s, all - 1) / per_row;
        *i = (s - *b * per_row) * 64 + lane;
        return u < each && s < all && *i < r.width;
    };
#pragma unroll
    for (int u = 0; u < kPieces; u++) {
        if (u >= each) break;
        int b, i;
        const bool in = place(u, &b, &i);
        const int entry = in ? r.table[b * r.table_row + i] : -1;
        x[u] = i >= r.kept(b) ? entry : -1;
    }
#pragma unroll
    for (int u = 0; u < kPieces; u++)
        if (u < each) n += __popcll(__ballot(r.is_page(x[u])));
    if (lane == 0) waves[wave] = n;
    __syncthreads();
    int at = have, total = have;
#pragma unroll
    for (int w = 0; w < kAllWaves; w++) {
        at += w < wave ? waves[w] : 0;
        total += waves[w];
    }
#pragma unroll
    for (int u = 0; u < kPieces; u++) {
        if (u >= each) break;
        const uint64_t back = __ballot(r.is_page(x[u]));
        const int to = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(back >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)back, 0));
        if (r.is_page(x[u]) && to < r.p.pages) r.p.free[to] = x[u];
        if (x[u] != -1) {
            int b, i;
            place(u, &b, &i);
            r.table[b * r.table_row + i] = -1;
        }
        at += __popcll(back);
    }
    if (threadIdx.x == 0) *r.p.count = min(total, r.p.pages);
}

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

// Larger tables, a workgroup to a row: how many pages it gives back, and then those
// behind what the rows before it do.
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
    __shared__ int waves[kWaves], found[kRows][kWaves];
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mine = r.counts[b];
    if (mine == 0 && b != r.batch - 1) return;
    int before = 0;
    for (int i = threadIdx.x; i < b; i += kThreads) before += r.counts[i];
    int at = *r.base + sum_of(before, waves);
    if (b == r.batch - 1 && threadIdx.x == 0) *r.p.count = min(at + mine, r.p.pages);
    if (mine == 0) return;
    int32_t* row = r.table + b * r.table_row;
    for (int first = r.kept(b); first < r.width; first += kRows * kThreads) {
        int x[kRows];
        uint64_t back[kRows];
#pragma unroll
        for (int u = 0; u < kRows; u++) {
            const int i = first + u * kThreads + threadIdx.x;
            x[u] = i < r.width ? row[i] : -1;
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kRows; u++) {
            back[u] = __ballot(r.is_page(x[u]));
            if (lane == 0) found[u][wave] = __popcll(back[u]);
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kRows; u++) {
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

// Whether `bytes` at a and n integers at b share memory.
bool overlap(const void* a, int64_t bytes, const int32_t* b, int64_t n) {
    return b && n > 0 && bytes > 0 && (uintptr_t)a < (uintptr_t)(b + n) && (uintptr_t)b < (uintptr_t)a + bytes;
}

bool one_launch(int table_width, int batch) {
    return (int64_t)((table_width + 63) / 64) * batch <= kAllWaves * kPieces;
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
    const struct { const void* at; int64_t bytes; } outs[] = {
        {slots, tokens * 8}, {positions, tokens * 4}, {filled, tokens * 4},
        {starts, 4 * ((int64_t)batch + 1)}, {new_lengths, 4 * (int64_t)batch}};
    const int64_t entries = batch ? table_row * (batch - 1) + table_width : 0;
    for (const auto& o : outs)
        if (overlap(o.at, o.bytes, lengths, batch) || overlap(o.at, o.bytes, fresh, batch) ||
            overlap(o.at, o.bytes, seen, batch) || overlap(o.at, o.bytes, table, entries) ||
            overlap(o.at, o.bytes, p->free, p->pages) || overlap(o.at, o.bytes, p->count, 1) ||
            overlap(o.at, o.bytes, p->ticket, 1))
            return RANS_EARG;
    const Extend e{*p, __builtin_ctz(p->page_size), table, table_row, table_width, lengths, fresh, seen, batch,
                   (int)tokens, slots, positions, filled, starts, new_lengths};
    const int64_t blocks = (tokens + kRows * kThreads - 1) / (kRows * kThreads);
    hipLaunchKernelGGL(extend_kernel, dim3(blocks ? (unsigned)blocks : 1), dim3(kThreads), (size_t)batch * 8, stream, e);
    return (int)hipGetLastError();
}

extern "C" int64_t vramc_pages_release_workspace(const vramc_pages* p, int table_width, int batch) {
    if (const int rc = check_table(p, table_width, table_width, batch)) return rc;
    return one_launch(table_width, batch) ? 0 : 4 * ((int64_t)batch + 1);
}

extern "C" int vramc_pages_release(const vramc_pages* p, int32_t* table, int64_t table_row,
                                   int table_width, const int32_t* lengths, int batch, void* workspace,
                                   int64_t workspace_bytes, hipStream_t stream) {
    if (const int rc = check_table(p, table_row, table_width, batch)) return rc;
    if (batch == 0 || table_width == 0) return 0;
    if (!table || !lengths) return RANS_EARG;
    const int64_t need = vramc_pages_release_workspace(p, table_width, batch);
    if (need && (!workspace || workspace_bytes < need)) return RANS_EWORKSPACE;
    if (need && (uintptr_t)workspace % 16) return RANS_EARG;
    auto* counts = static_cast<int32_t*>(workspace);
    const Release r{*p, __builtin_ctz(p->page_size), table, table_row, table_width, lengths, batch, counts,
                    counts + batch};
    if (!need) {
        hipLaunchKernelGGL(release_kernel, dim3(1), dim3(kAll), 0, stream, r);
        return (int)hipGetLastError();
    }
    hipLaunchKernelGGL(release_count_kernel, dim3((unsigned)batch), dim3(kThreads), 0, stream, r);
    if (const int rc = (int)hipGetLastError()) return rc;
    hipLaunchKernelGGL(release_rows_kernel, dim3((unsigned)batch), dim3(kThreads), 0, stream, r);
    return (int)hipGetLastError();
}
