// New tokens' keys and values into the pages of a cache, and back.
//
// Both are passes over their bytes: one thread takes eight values of a token's
// head, 16 bytes of a 16-bit type, so that a wave reads and writes contiguous
// rows.  In 4-bit storage four neighbouring threads hold a block of 32 and
// agree on its scale.
#include "kv_device.h"

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 8;  // values of a thread

// floor(log2(a)) for a finite a > 0, subnormals included.
__device__ __forceinline__ int floor_log2(float a) {
    const int e = (int)(__float_as_uint(a) >> 23);
    return e ? e - 127 : -118 - __clz((int)__float_as_uint(a));
}

// The code nearest to y, ties to the even one: the number of midpoints below
// |y|, of which every second one belongs to the code above it.
__device__ __forceinline__ uint32_t mx_code(float y) {
    const float a = fabsf(y);
    const uint32_t n = (a > 0.25f) + (a >= 0.75f) + (a > 1.25f) + (a >= 1.75f) + (a > 2.5f) +
                       (a >= 3.5f) + (a > 5.f);
    return n | (__float_as_uint(y) >> 31 << 3);
}

template <typename T, bool MX, bool WIDE>
__global__ void __launch_bounds__(kThreads)
    kv_append_kernel(vramc_kv_cache c, const T* __restrict__ k, int64_t k_token, int64_t k_head,
                     const T* __restrict__ v, int64_t v_token, int64_t v_head,
                     const int64_t* __restrict__ slots, const int32_t* __restrict__ positions,
                     int64_t tokens) {
    const int per_row = c.head_dim / kPer;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t row = i / per_row;  // token and head
    const int seg = (int)(i - row * per_row);
    const int64_t t = row / c.kv_heads;
    const int h = (int)(row - t * c.kv_heads);
    // threads of a block of 32 columns share a token: they leave together
    if (t >= tokens) return;
    const int64_t slot = slots[t];
    if (slot < 0 || slot >= (int64_t)c.pages * c.page_size) return;
    const bool values = blockIdx.y;
    const T* in = values ? v + t * v_token + h * v_head : k + t * k_token + h * k_head;
    const int64_t page = slot / c.page_size;
    const int64_t at = (page * c.kv_heads + h) * c.page_size + (slot - page * c.page_size);
    vec<T, kPer> x;
    if (WIDE) {
        x = *reinterpret_cast<const vec<T, kPer>*>(in + seg * kPer);
    } else {
#pragma unroll
        for (int j = 0; j < kPer; j++) x[j] = in[seg * kPer + j];
    }
    if (!MX) {
        auto* out = static_cast<T*>(values ? c.v : c.k) + at * c.head_dim + seg * kPer;
        *reinterpret_cast<vec<T, kPer>*>(out) = x;
    } else {
        float most = 0.f;
        bool bad = false;
#pragma unroll
        for (int j = 0; j < kPer; j++) {
            const float a = fabsf((float)x[j]);
            bad |= !(a <= __FLT_MAX__);
            most = fmaxf(most, a);
        }
        if (bad) most = __builtin_inff();
        most = fmaxf(most, __shfl_xor(most, 1));
        most = fmaxf(most, __shfl_xor(most, 2));
        bad = most > __FLT_MAX__;
        const int e = most == 0.f || bad ? -127 : max(floor_log2(most) - 2, -127);
        uint32_t codes = 0;
        if (!bad) {
            const float unit = __uint_as_float((uint32_t)(127 - e) << 23);  // 2^-e
#pragma unroll
            for (int j = 0; j < kPer; j++) codes |= mx_code((float)x[j] * unit) << 4 * j;
        }
        auto* out = static_cast<uint32_t*>(values ? c.v : c.k) + at * per_row + seg;
        *out = codes;
        if (seg % 4 == 0)
            (values ? c.v_scale : c.k_scale)[at * (c.head_dim / kMxBlock) + seg / 4] =
                bad ? 255 : (uint8_t)(e + 127);
    }
    if (c.mass && !values && seg == 0) {
        c.mass[at] = 0.f;
        c.position[at] = positions[t];
    }
}

template <typename T, bool MX>
__global__ void __launch_bounds__(kThreads)
    kv_read_kernel(vramc_kv_cache c, const int64_t* __restrict__ slots, T* __restrict__ k,
                   T* __restrict__ v, int64_t tokens) {
    const int per_row = c.head_dim / kPer;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    const int64_t row = i / per_row;
    const int seg = (int)(i - row * per_row);
    const int64_t t = row / c.kv_heads;
    const int h = (int)(row - t * c.kv_heads);
    if (t >= tokens) return;
    const bool values = blockIdx.y;
    const int64_t slot = slots[t];
    vec<T, kPer> x = {};
    if (slot >= 0 && slot < (int64_t)c.pages * c.page_size) {
        const int64_t page = slot / c.page_size;
        const int64_t at = (page * c.kv_heads + h) * c.page_size + (slot - page * c.page_size);
        const void* held = values ? c.v : c.k;
        if (!MX) {
            x = *reinterpret_cast<const vec<T, kPer>*>(static_cast<const T*>(held) +
                                                       at * c.head_dim + seg * kPer);
        } else {
            const uint32_t codes = static_cast<const uint32_t*>(held)[at * per_row + seg];
            const float unit = mx_power((values ? c.v_scale : c.k_scale)[
                at * (c.head_dim / kMxBlock) + seg / 4]);
#pragma unroll
            for (int j = 0; j < kPer; j++) x[j] = (T)(mx_value(codes >> 4 * j & 15) * unit);
        }
    }
    *reinterpret_cast<vec<T, kPer>*>((values ? v : k) + i * kPer) = x;
}

// Whether rows at these strides can be read eight values at a time.
template <typename T>
bool wide(const void* p, int64_t token, int64_t head) {
    return ((uintptr_t)p | (uintptr_t)(token * (int64_t)sizeof(T)) |
            (uintptr_t)(head * (int64_t)sizeof(T))) % (kPer * sizeof(T)) == 0;
}

template <typename T, bool MX>
int append(const vramc_kv_cache& c, const void* k, int64_t k_token, int64_t k_head, const void* v,
           int64_t v_token, int64_t v_head, const int64_t* slots, const int32_t* positions,
           int64_t tokens, dim3 grid, hipStream_t stream) {
    const auto *kp = static_cast<const T*>(k), *vp = static_cast<const T*>(v);
    if (wide<T>(k, k_token, k_head) && wide<T>(v, v_token, v_head))
        hipLaunchKernelGGL((kv_append_kernel<T, MX, true>), grid, dim3(kThreads), 0, stream, c, kp,
                           k_token, k_head, vp, v_token, v_head, slots, positions, tokens);
    else
        hipLaunchKernelGGL((kv_append_kernel<T, MX, false>), grid, dim3(kThreads), 0, stream, c, kp,
                           k_token, k_head, vp, v_token, v_head, slots, positions, tokens);
    return (int)hipGetLastError();
}

template <typename T, bool MX>
int read(const vramc_kv_cache& c, const int64_t* slots, int64_t tokens, void* k, void* v,
         dim3 grid, hipStream_t stream) {
    hipLaunchKernelGGL((kv_read_kernel<T, MX>), grid, dim3(kThreads), 0, stream, c, slots,
                       static_cast<T*>(k), static_cast<T*>(v), tokens);
    return (int)hipGetLastError();
}

// Workgroups of `tokens` rows, 0 for more than a grid holds.
int64_t blocks(const vramc_kv_cache& c, int64_t tokens) {
    const int64_t row = (int64_t)c.kv_heads * (c.head_dim / kPer);
    if (tokens > ((int64_t)INT32_MAX * kThreads) / row) return 0;
    return (tokens * row + kThreads - 1) / kThreads;
}

}  // namespace

extern "C" int vramc_kv_append(const vramc_kv_cache* c, const void* k, int64_t k_token,
                               int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                               const int64_t* slots, const int32_t* positions, int64_t tokens,
                               hipStream_t stream) {
    if (const int rc = check_cache(c)) return rc;
    if (tokens < 0) return RANS_EARG;
    if (tokens == 0) return 0;
    if (!k || !v || !slots || (c->mass && !positions)) return RANS_EARG;
    const int64_t n = blocks(*c, tokens);
    if (!n) return RANS_EARG;
    const dim3 grid((unsigned)n, 2);
    const auto go = [&](auto fn) {
        return fn(*c, k, k_token, k_head, v, v_token, v_head, slots, positions, tokens, grid, stream);
    };
    if (c->dtype == RANS_X_F32) return go(append<float, false>);
    if (c->dtype == RANS_X_BF16) return c->mx ? go(append<__bf16, true>) : go(append<__bf16, false>);
    return c->mx ? go(append<_Float16, true>) : go(append<_Float16, false>);
}

extern "C" int vramc_kv_read(const vramc_kv_cache* c, const int64_t* slots, int64_t tokens,
                             void* k_out, void* v_out, hipStream_t stream) {
    if (const int rc = check_cache(c)) return rc;
    if (tokens < 0) return RANS_EARG;
    if (tokens == 0) return 0;
    if (!slots || !k_out || !v_out || ((uintptr_t)k_out | (uintptr_t)v_out) % 32) return RANS_EARG;
    const int64_t n = blocks(*c, tokens);
    if (!n) return RANS_EARG;
    const dim3 grid((unsigned)n, 2);
    const auto go = [&](auto fn) { return fn(*c, slots, tokens, k_out, v_out, grid, stream); };
    if (c->dtype == RANS_X_F32) return go(read<float, false>);
    if (c->dtype == RANS_X_BF16) return c->mx ? go(read<__bf16, true>) : go(read<__bf16, false>);
    return c->mx ? go(read<_Float16, true>) : go(read<_Float16, false>);
}
