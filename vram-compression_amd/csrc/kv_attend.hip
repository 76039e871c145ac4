// Attention of one new token of each sequence over a paged cache.
//
// The simple form: one workgroup for a query head of a sequence goes through
// the tokens 256 at a time, one thread a token for the scores, one thread a
// column for the values, with a running maximum and sum.
#include "kv_device.h"

namespace {

constexpr int kThreads = 256;

struct Attend {
    vramc_kv_cache c;
    const void* q;
    int64_t q_seq, q_head;
    int q_heads;
    const int32_t* table;
    int64_t table_row;
    int table_width;
    const int32_t* lengths;
    int batch;
    float scale;
    void* out;
    float* scores;  // [batch * q_heads][tokens], where weights are tracked
    float2* sums;   // [batch * q_heads]: maximum and sum
};

template <typename T, bool MX>
__device__ float held(const void* p, const uint8_t* scale, int64_t at, int dim, int d) {
    if (!MX) return (float)static_cast<const T*>(p)[at * dim + d];
    const uint32_t b = static_cast<const uint8_t*>(p)[at * (dim / 2) + d / 2];
    return mx_value(d & 1 ? b >> 4 : b & 15) * mx_power(scale[at * (dim / kMxBlock) + d / kMxBlock]);
}

__device__ float block_max(float x, float* buf) {
    buf[threadIdx.x] = x;
    __syncthreads();
    for (int n = kThreads / 2; n; n /= 2) {
        if ((int)threadIdx.x < n) buf[threadIdx.x] = fmaxf(buf[threadIdx.x], buf[threadIdx.x + n]);
        __syncthreads();
    }
    const float r = buf[0];
    __syncthreads();
    return r;
}

__device__ float block_sum(float x, float* buf) {
    buf[threadIdx.x] = x;
    __syncthreads();
    for (int n = kThreads / 2; n; n /= 2) {
        if ((int)threadIdx.x < n) buf[threadIdx.x] += buf[threadIdx.x + n];
        __syncthreads();
    }
    const float r = buf[0];
    __syncthreads();
    return r;
}

template <typename T, bool MX>
__global__ void __launch_bounds__(kThreads) attend_kernel(Attend a) {
    __shared__ float q[256], p[kThreads], buf[kThreads];
    __shared__ int64_t place[kThreads];
    const int b = blockIdx.x / a.q_heads, head = blockIdx.x % a.q_heads;
    const int h = head / (a.q_heads / a.c.kv_heads), dim = a.c.head_dim, ps = a.c.page_size;
    const int64_t bound = (int64_t)a.table_width * ps;
    const int n = (int)min((int64_t)max(a.lengths[b], 0), bound);
    const int d = threadIdx.x;
    if (d < dim) q[d] = (float)static_cast<const T*>(a.q)[b * a.q_seq + head * a.q_head + d];
    __syncthreads();
    float m = -__builtin_inff(), l = 0.f, o = 0.f;
    for (int first = 0; first < n; first += kThreads) {
        const int j = first + threadIdx.x;
        float s = -__builtin_inff();
        int64_t at = -1;
        if (j < n) {
            const int page = a.table[b * a.table_row + j / ps];
            if (page >= 0 && page < a.c.pages) {
                at = ((int64_t)page * a.c.kv_heads + h) * ps + j % ps;
                float sum = 0.f;
                for (int i = 0; i < dim; i++)
                    sum += q[i] * held<T, MX>(a.c.k, a.c.k_scale, at, dim, i);
                s = sum * a.scale;
            }
            if (a.scores) a.scores[blockIdx.x * bound + j] = s;
        }
        place[threadIdx.x] = at;
        const float top = fmaxf(m, block_max(s, buf));
        const float from = top == -__builtin_inff() ? 0.f : top;
        const float w = at < 0 ? 0.f : expf(s - from);
        p[threadIdx.x] = w;
        const float keep = m == -__builtin_inff() ? 0.f : expf(m - from);
        l = l * keep + block_sum(w, buf);
        o *= keep;
        m = top;
        if (d < dim)
            for (int i = 0; i < kThreads; i++)
                if (place[i] >= 0) o += p[i] * held<T, MX>(a.c.v, a.c.v_scale, place[i], dim, d);
        __syncthreads();
    }
    if (d < dim)
        static_cast<T*>(a.out)[(int64_t)blockIdx.x * dim + d] = (T)(l == 0.f ? 0.f : o / l);
    if (a.sums && d == 0) a.sums[blockIdx.x] = make_float2(m, l);
}

// mass[token] += sum of the weights over the kv head's query heads.
__global__ void __launch_bounds__(kThreads) mass_kernel(Attend a) {
    const int b = blockIdx.y / a.c.kv_heads, h = blockIdx.y % a.c.kv_heads, ps = a.c.page_size;
    const int64_t bound = (int64_t)a.table_width * ps;
    const int64_t j = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (j >= a.lengths[b] || j >= bound) return;
    const int page = a.table[b * a.table_row + j / ps];
    if (page < 0 || page >= a.c.pages) return;
    const int group = a.q_heads / a.c.kv_heads;
    float w = 0.f;
    for (int g = 0; g < group; g++) {
        const int64_t row = (int64_t)b * a.q_heads + h * group + g;
        const float2 ml = a.sums[row];
        if (ml.y != 0.f) w += expf(a.scores[row * bound + j] - (ml.x == -__builtin_inff() ? 0.f : ml.x)) / ml.y;
    }
    atomicAdd(&a.c.mass[((int64_t)page * a.c.kv_heads + h) * ps + j % ps], w);
}

template <typename T, bool MX>
int attend(const Attend& a, hipStream_t stream) {
    hipLaunchKernelGGL((attend_kernel<T, MX>), dim3(a.batch * a.q_heads), dim3(kThreads), 0, stream, a);
    if (const int rc = (int)hipGetLastError()) return rc;
    if (!a.scores) return 0;
    const int64_t bound = (int64_t)a.table_width * a.c.page_size;
    hipLaunchKernelGGL(mass_kernel, dim3((unsigned)((bound + kThreads - 1) / kThreads), a.batch * a.c.kv_heads),
                       dim3(kThreads), 0, stream, a);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" int64_t vramc_kv_attend_workspace(const vramc_kv_cache* c, int q_heads, int table_width,
                                             int batch, int track) {
    if (const int rc = check_cache(c)) return rc;
    if (q_heads <= 0 || q_heads % c->kv_heads || table_width < 0 || batch < 0) return RANS_EARG;
    if ((int64_t)table_width * c->page_size > kMaxTokens || (int64_t)batch * q_heads > 65535) return RANS_EARG;
    if (!track) return 0;
    return (int64_t)batch * q_heads * (8 + 4 * (int64_t)table_width * c->page_size);
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
    Attend a{*c, q, q_seq, q_head, q_heads, table, table_row, table_width, lengths, batch, scale,
             out, nullptr, nullptr};
    if (track && table_width) {
        a.sums = static_cast<float2*>(workspace);
        a.scores = static_cast<float*>(workspace) + 2 * (int64_t)batch * q_heads;
    }
    if (c->dtype == RANS_X_F32) return attend<float, false>(a, stream);
    if (c->dtype == RANS_X_BF16)
        return c->mx ? attend<__bf16, true>(a, stream) : attend<__bf16, false>(a, stream);
    return c->mx ? attend<_Float16, true>(a, stream) : attend<_Float16, false>(a, stream);
}
