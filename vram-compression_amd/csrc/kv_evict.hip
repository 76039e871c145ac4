// Eviction of a cache's tokens by accumulated weight.
//
// A kv head of a sequence ranks its tokens by a 32-bit key that sorts as the
// order of eviction does.  The budget-th largest key is found by radix
// selection, eight bits at a time; every token above it is kept, and of those
// equal to it as many as there is room for, lowest index first.  What moves
// where is then two ordered lists, and moving is a copy of rows that are all
// different places.
#include "kv_device.h"

namespace {

constexpr int kSelect = 1024;  // threads that select
constexpr int kMove = 256;     // threads that move

struct Evict {
    vramc_kv_cache c;
    const int32_t* table;
    int64_t table_row;
    int table_width;
    const int32_t *lengths, *seen;
    int batch, budget, recent;
    const int32_t* into;
    int64_t into_row;
    int into_width;
    int32_t* new_lengths;
    int32_t *from, *to, *count;  // [batch * kv_heads][most] places, and how many
    int most;
};

// The place of token j: slot of the cache for a kv head, -1 for none.
__device__ __forceinline__ int64_t place(const Evict& e, const int32_t* row, int h, int j) {
    const int page = row[j / e.c.page_size];
    if (page < 0 || page >= e.c.pages) return -1;
    return ((int64_t)page * e.c.kv_heads + h) * e.c.page_size + j % e.c.page_size;
}

// Sorts as the order in which tokens are kept: 0 for a token that is nowhere,
// the mass's bits made monotonic (NaN as -infinity), all ones for a recent one.
__device__ __forceinline__ uint32_t rank_of(const Evict& e, int64_t at, int from_position) {
    if (at < 0) return 0;
    if (e.c.position[at] >= from_position) return 0xffffffffu;
    float m = e.c.mass[at];
    if (m != m) m = -__builtin_inff();
    const uint32_t bits = __float_as_uint(m + 0.f);  // -0 as 0
    return bits >> 31 ? ~bits : bits | 0x80000000u;
}

// Exclusive sum over the workgroup's threads; total in *sum.
__device__ int scan(int x, int* buf, int* sum) {
    const int t = threadIdx.x;
    buf[t] = x;
    __syncthreads();
    for (int n = 1; n < kSelect; n *= 2) {
        const int y = t >= n ? buf[t - n] : 0;
        __syncthreads();
        buf[t] += y;
        __syncthreads();
    }
    *sum = buf[kSelect - 1];
    const int before = buf[t] - x;
    __syncthreads();
    return before;
}

__global__ void __launch_bounds__(kSelect) select_kernel(Evict e) {
    __shared__ int hist[256], buf[kSelect], found[2];
    const int b = blockIdx.x / e.c.kv_heads, h = blockIdx.x % e.c.kv_heads;
    const int bound = e.table_width * e.c.page_size;
    const int n = min(max(e.lengths[b], 0), bound);
    const int32_t* row = e.table + b * e.table_row;
    const int64_t from_position = (int64_t)e.seen[b] - e.recent;
    const int recent = (int)max(from_position, (int64_t)INT32_MIN);
    if (h == 0 && threadIdx.x == 0) e.new_lengths[b] = min(n, e.budget);
    int32_t* from = e.from + (int64_t)blockIdx.x * e.most;
    int32_t* to = e.to + (int64_t)blockIdx.x * e.most;
    if (n <= e.budget) {  // everything is kept
        if (threadIdx.x == 0) e.count[blockIdx.x] = e.into ? n : 0;
        if (e.into)
            for (int j = threadIdx.x; j < n; j += kSelect) from[j] = to[j] = j;
        return;
    }
    uint32_t above = 0;     // the digits found so far
    int room = e.budget;    // tokens to keep of those that share them
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kSelect) hist[i] = 0;
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += kSelect) {
            const uint32_t r = rank_of(e, place(e, row, h, j), recent);
            if (shift == 24 || r >> (shift + 8) == above >> (shift + 8))
                atomicAdd(&hist[r >> shift & 255], 1);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int digit = 255, left = room;
            while (hist[digit] < left) left -= hist[digit--];
            found[0] = digit;
            found[1] = left;
        }
        __syncthreads();
        above |= (uint32_t)found[0] << shift;
        room = found[1];
        __syncthreads();
    }
    // `above` is the budget-th largest rank, `room` of its tokens are kept
    int ties = 0, holes = 0, kept_above = 0, kept = 0;
    for (int first = 0; first < n; first += kSelect) {
        const int j = first + threadIdx.x;
        const uint32_t r = j < n ? rank_of(e, place(e, row, h, j), recent) : 0;
        int sum;
        const bool tie = j < n && r == above;
        const int tied = ties + scan(tie, buf, &sum);
        ties += sum;
        const bool keep = j < n && (r > above || (tie && tied < room));
        if (e.into) {
            const int i = kept + scan(keep, buf, &sum);
            kept += sum;
            if (keep) from[i] = j, to[i] = i;
        } else {
            const bool hole = j < e.budget && !keep;
            int i = holes + scan(hole, buf, &sum);
            holes += sum;
            if (hole) to[i] = j;
            const bool moves = keep && j >= e.budget;
            i = kept_above + scan(moves, buf, &sum);
            kept_above += sum;
            if (moves) from[i] = j;
        }
    }
    if (threadIdx.x == 0) e.count[blockIdx.x] = e.into ? kept : kept_above;
}

// One wave moves a token of a kv head.
__global__ void __launch_bounds__(kMove) move_kernel(Evict e) {
    const int group = blockIdx.y, b = group / e.c.kv_heads, h = group % e.c.kv_heads;
    const int i = blockIdx.x * (kMove / 64) + threadIdx.x / 64, lane = threadIdx.x & 63;
    if (i >= e.count[group]) return;
    const int64_t from = place(e, e.table + b * e.table_row, h, e.from[(int64_t)group * e.most + i]);
    const int64_t to = place(e, e.into ? e.into + b * e.into_row : e.table + b * e.table_row, h,
                             e.to[(int64_t)group * e.most + i]);
    if (from < 0 || to < 0) return;
    const int size = e.c.dtype == RANS_X_F32 ? 4 : 2;
    const int bytes = e.c.mx ? e.c.head_dim / 2 : e.c.head_dim * size;
    for (int which = 0; which < 2; which++) {
        auto* p = static_cast<uint32_t*>(which ? e.c.v : e.c.k);
        for (int j = lane; j < bytes / 4; j += 64) p[to * (bytes / 4) + j] = p[from * (bytes / 4) + j];
        if (e.c.mx && lane < e.c.head_dim / kMxBlock) {
            uint8_t* s = which ? e.c.v_scale : e.c.k_scale;
            s[to * (e.c.head_dim / kMxBlock) + lane] = s[from * (e.c.head_dim / kMxBlock) + lane];
        }
    }
    if (lane == 0) {
        e.c.mass[to] = e.c.mass[from];
        e.c.position[to] = e.c.position[from];
    }
}

// Tokens of a kv head that one call can move.
int64_t most_moves(const vramc_kv_cache& c, int table_width, int budget, bool into) {
    const int64_t bound = (int64_t)table_width * c.page_size;
    if (into) return budget < bound ? budget : bound;
    const int64_t over = bound > budget ? bound - budget : 0;
    return budget < over ? budget : over;
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
    const int64_t heads = (int64_t)batch * c->kv_heads;
    auto* count = static_cast<int32_t*>(workspace);
    Evict e{*c, table, table_row, table_width, lengths, seen, batch, budget, recent, into, into_row,
            into_width, new_lengths, count + heads, count + heads + heads * most, count, (int)most};
    hipLaunchKernelGGL(select_kernel, dim3((unsigned)heads), dim3(kSelect), 0, stream, e);
    if (const int rc = (int)hipGetLastError()) return rc;
    if (!most) return 0;
    const int rows = kMove / 64;
    hipLaunchKernelGGL(move_kernel, dim3((unsigned)((most + rows - 1) / rows), (unsigned)heads),
                       dim3(kMove), 0, stream, e);
    return (int)hipGetLastError();
}
