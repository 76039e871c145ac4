// New tokens' keys and values into the pages of a cache, and back.
//
// Both are passes over their bytes, and HBM bounds them: 32768 tokens of 8 heads
// of 128 columns into 4-bit pages 37.8 us (4.6 TB/s; a large copy reaches 5.0), in
// bf16 53.9 us (5.0 TB/s).  Back, behind such an append, whose bytes fill the
// caches, 32.0 us (5.3 TB/s, mostly writes) and 45.6 us (5.9 TB/s), and 25.5 and
// 42.4 us again and again.  One token of each of 16 sequences 2.5 and 2.0 us.
//
// One thread takes eight values of a token's head, 16 bytes of a 16-bit type; a
// workgroup takes neighbouring tokens of one head, whose rows lie behind each
// other in a page, so that also the quarter as long rows of 4-bit codes are
// written whole lines at a time.  Workgroups of 128 to 1024 threads, the heads of
// some tokens on one XCD and two rows a thread take the same time; heads behind
// each other in time cost 46.5 us in place of 38.8 (8192 tokens of 32 heads).  In
// 4-bit storage four neighbouring threads hold a block of 32 and agree on its
// scale; codes are made by the hardware's conversion, which rounds to the nearest,
// ties to the even code, and saturates.
#include "kv_device.h"

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 8;  // values of a thread

// Eight values where they lie in a cache, whose tensors are aligned to 16 bytes: as
// one vector, eight floats would promise 32.
template <typename T>
struct Lying {
    vec<uint32_t, 4> part[kPer * sizeof(T) / 16];
};

// The largest magnitude of eight values, as the bits of a float: magnitudes of a
// float format sort as their bits do, infinity and NaN above all.
template <typename T>
__device__ __forceinline__ uint32_t largest(vec<T, kPer> x) {
    const auto bits = __builtin_bit_cast(vec<uint16_t, kPer>, x) & (uint16_t)0x7fff;
    const auto a = __builtin_elementwise_max(bits.lo, bits.hi);
    const auto b = __builtin_elementwise_max(a.lo, a.hi);
    return __float_as_uint((float)__builtin_bit_cast(T, (uint16_t)max(b[0], b[1])));
}

// Eight codes of x / unit, unit a power of two.
template <typename T>
__device__ __forceinline__ uint32_t mx_codes(vec<T, kPer> x, float unit) {
    const vec<T, 2> a = x.s01, b = x.s23, c = x.s45, d = x.s67;
    uint32_t r = 0;
    if constexpr (std::is_same_v<T, __bf16>) {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, a, unit, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, b, unit, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, c, unit, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, d, unit, 3);
    } else {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, a, unit, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, b, unit, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, c, unit, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, d, unit, 3);
    }
}

// What a thread's row is: a token of a head, and where it lies in the cache.
struct Row {
    int64_t token, at;
    int head;
    bool there;
};
__device__ __forceinline__ Row row_of(const vramc_kv_cache& c, int page_shift,
                                      const int64_t* __restrict__ slots, int64_t tokens) {
    Row r;
    const uint32_t block = blockIdx.x / c.kv_heads;
    r.token = (int64_t)block * blockDim.y + threadIdx.y;
    r.head = blockIdx.x - block * c.kv_heads;
    const int64_t slot = r.token < tokens ? slots[r.token] : -1;
    r.there = slot >= 0 && slot < (int64_t)c.pages << page_shift;
    r.at = (((slot >> page_shift) * c.kv_heads + r.head) << page_shift) + (slot & (c.page_size - 1));
    return r;
}

// Eight values of a row of the cache, written past the caches, which the tokens
// of a long append would only pass through (32768 tokens of 8 heads of 128
// columns in bf16 53.2 us against 55.1, in 4 bits 38.9 against 40.4).
template <typename T, bool MX>
__device__ __forceinline__ void store(vec<T, kPer> x, void* held, uint8_t* scales, int64_t at, int per_row,
                                      int seg) {
    if constexpr (!MX) {
        const auto from = __builtin_bit_cast(Lying<T>, x);
        auto* to = static_cast<Lying<T>*>(held) + at * per_row + seg;
#pragma unroll
        for (size_t i = 0; i < sizeof(T) / 2; i++) __builtin_nontemporal_store(from.part[i], &to->part[i]);
    } else {
        // a block's threads are four neighbours of a wave
        uint32_t most = largest(x);
        most = max(most, (uint32_t)__shfl_xor((int)most, 1));
        most = max(most, (uint32_t)__shfl_xor((int)most, 2));
        // the scale's byte, floor(log2(most)) - 2 + 127, from the exponent's bits
        const int bits = (int)(most >> 23);
        const int byte = bits == 255 ? 255 : max(bits - 2, 0);
        const uint32_t codes = mx_codes(x, __uint_as_float((uint32_t)byte << 23));
        __builtin_nontemporal_store(byte == 255 ? 0u : codes, static_cast<uint32_t*>(held) + at * per_row + seg);
        if (seg % 4 == 0) scales[at * (per_row / 4) + seg / 4] = (uint8_t)byte;
    }
}

// Eight values of a row of the cache, read.
template <typename T, bool MX>
struct Held {
    vec<T, kPer> x;
    uint32_t codes, scale;
    __device__ __forceinline__ void load(const void* held, const uint8_t* scales, int64_t at, int per_row,
                                         int seg) {
        if constexpr (!MX) {
            x = __builtin_bit_cast(vec<T, kPer>, static_cast<const Lying<T>*>(held)[at * per_row + seg]);
        } else {
            codes = static_cast<const uint32_t*>(held)[at * per_row + seg];
            scale = scales[at * (per_row / 4) + seg / 4];
        }
    }
    __device__ __forceinline__ vec<T, kPer> values() const {
        if constexpr (!MX) {
            return x;
        } else {
            vec<uint32_t, 4> pairs;
#pragma unroll
            for (int i = 0; i < 4; i++) pairs[i] = mx_pair_at<T>(codes, scale, i);
            return __builtin_bit_cast(vec<T, kPer>, pairs);
        }
    }
};

template <typename T, bool WIDE>
__device__ __forceinline__ vec<T, kPer> load(const T* in) {
    if constexpr (WIDE) return *reinterpret_cast<const vec<T, kPer>*>(in);
    vec<T, kPer> x;
#pragma unroll
    for (int j = 0; j < kPer; j++) x[j] = in[j];
    return x;
}

template <typename T, bool MX, bool WIDE>
__global__ void __launch_bounds__(kThreads)
    kv_append_kernel(vramc_kv_cache c, int page_shift, const T* __restrict__ k, int64_t k_token,
                     int64_t k_head, const T* __restrict__ v, int64_t v_token, int64_t v_head,
                     const int64_t* __restrict__ slots, const int32_t* __restrict__ positions,
                     int64_t tokens) {
    const int per_row = blockDim.x, seg = threadIdx.x;
    const Row r = row_of(c, page_shift, slots, tokens);
    if (r.token >= tokens) return;
    // before the slot is known, so that one wait covers both
    const auto x = load<T, WIDE>(k + r.token * k_token + r.head * k_head + seg * kPer);
    const auto y = load<T, WIDE>(v + r.token * v_token + r.head * v_head + seg * kPer);
    if (!r.there) return;  // the threads of a block of 32 columns share a row
    store<T, MX>(x, c.k, c.k_scale, r.at, per_row, seg);
    store<T, MX>(y, c.v, c.v_scale, r.at, per_row, seg);
    if (c.mass && seg == 0) {
        c.mass[r.at] = 0.f;
        c.position[r.at] = positions[r.token];
    }
}

template <typename T, bool MX>
__global__ void __launch_bounds__(kThreads)
    kv_read_kernel(vramc_kv_cache c, int page_shift, const int64_t* __restrict__ slots,
                   T* __restrict__ k, T* __restrict__ v, int64_t tokens) {
    const int per_row = blockDim.x, seg = threadIdx.x;
    const Row r = row_of(c, page_shift, slots, tokens);
    if (r.token >= tokens) return;
    vec<T, kPer> x = {}, y = {};
    if (r.there) {
        Held<T, MX> kh, vh;
        kh.load(c.k, c.k_scale, r.at, per_row, seg);
        vh.load(c.v, c.v_scale, r.at, per_row, seg);
        x = kh.values();
        y = vh.values();
    }
    const int64_t to = (r.token * c.kv_heads + r.head) * per_row + seg;
    auto *kp = reinterpret_cast<vec<T, kPer>*>(k) + to, *vp = reinterpret_cast<vec<T, kPer>*>(v) + to;
    // From 4-bit pages nearly all traffic is these stores: past the caches, 32768
    // tokens of 8 heads of 128 columns, again and again, take 26.0 us against 31.4.
    // Where as much is read as written it is the other way round (48.9 us against
    // 42.4).
    if constexpr (MX) {
        __builtin_nontemporal_store(x, kp);
        __builtin_nontemporal_store(y, vp);
    } else {
        *kp = x;
        *vp = y;
    }
}

// Whether rows at these strides can be read eight values at a time.
template <typename T>
bool wide(const void* p, int64_t token, int64_t head) {
    return ((uintptr_t)p | (uintptr_t)(token * (int64_t)sizeof(T)) |
            (uintptr_t)(head * (int64_t)sizeof(T))) % (kPer * sizeof(T)) == 0;
}

// Workgroups of whole rows of one head, neighbouring tokens each, the heads of
// a token next to each other in time, as they lie in memory; 0 for too many.
struct Shape {
    dim3 grid, block;
};
Shape shape_of(const vramc_kv_cache& c, int64_t tokens) {
    const int per_row = c.head_dim / kPer, rows = kThreads / per_row;
    const int64_t n = (tokens + rows - 1) / rows * c.kv_heads;
    return {dim3(n > kMaxThreads / kThreads ? 0 : (unsigned)n), dim3((unsigned)per_row, (unsigned)rows)};
}

template <typename T, bool MX>
int append(const vramc_kv_cache& c, const void* k, int64_t k_token, int64_t k_head, const void* v,
           int64_t v_token, int64_t v_head, const int64_t* slots, const int32_t* positions,
           int64_t tokens, hipStream_t stream) {
    const auto *kp = static_cast<const T*>(k), *vp = static_cast<const T*>(v);
    const Shape s = shape_of(c, tokens);
    if (!s.grid.x) return RANS_EARG;
    const int shift = __builtin_ctz(c.page_size);
    if (wide<T>(k, k_token, k_head) && wide<T>(v, v_token, v_head))
        hipLaunchKernelGGL((kv_append_kernel<T, MX, true>), s.grid, s.block, 0, stream, c, shift, kp,
                           k_token, k_head, vp, v_token, v_head, slots, positions, tokens);
    else
        hipLaunchKernelGGL((kv_append_kernel<T, MX, false>), s.grid, s.block, 0, stream, c, shift, kp,
                           k_token, k_head, vp, v_token, v_head, slots, positions, tokens);
    return (int)hipGetLastError();
}

template <typename T, bool MX>
int read(const vramc_kv_cache& c, const int64_t* slots, int64_t tokens, void* k, void* v,
         hipStream_t stream) {
    const Shape s = shape_of(c, tokens);
    if (!s.grid.x) return RANS_EARG;
    hipLaunchKernelGGL((kv_read_kernel<T, MX>), s.grid, s.block, 0, stream, c,
                       __builtin_ctz(c.page_size), slots, static_cast<T*>(k), static_cast<T*>(v), tokens);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" int vramc_kv_append(const vramc_kv_cache* c, const void* k, int64_t k_token,
                               int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                               const int64_t* slots, const int32_t* positions, int64_t tokens,
                               hipStream_t stream) {
    if (const int rc = check_cache(c)) return rc;
    if (tokens < 0 || tokens > INT64_MAX / 65536) return RANS_EARG;
    if (tokens == 0) return 0;
    if (!k || !v || !slots || (c->mass && !positions)) return RANS_EARG;
    const auto go = [&](auto fn) {
        return fn(*c, k, k_token, k_head, v, v_token, v_head, slots, positions, tokens, stream);
    };
    if (c->dtype == RANS_X_F32) return go(append<float, false>);
    if (c->dtype == RANS_X_BF16) return c->mx ? go(append<__bf16, true>) : go(append<__bf16, false>);
    return c->mx ? go(append<_Float16, true>) : go(append<_Float16, false>);
}

extern "C" int vramc_kv_read(const vramc_kv_cache* c, const int64_t* slots, int64_t tokens,
                             void* k_out, void* v_out, hipStream_t stream) {
    if (const int rc = check_cache(c)) return rc;
    if (tokens < 0 || tokens > INT64_MAX / 65536) return RANS_EARG;
    if (tokens == 0) return 0;
    if (!slots || !k_out || !v_out || ((uintptr_t)k_out | (uintptr_t)v_out) % 32) return RANS_EARG;
    const auto go = [&](auto fn) { return fn(*c, slots, tokens, k_out, v_out, stream); };
    if (c->dtype == RANS_X_F32) return go(read<float, false>);
    if (c->dtype == RANS_X_BF16) return c->mx ? go(read<__bf16, true>) : go(read<__bf16, false>);
    return c->mx ? go(read<_Float16, true>) : go(read<_Float16, false>);
}
