// What the key-value cache's kernels share: the 4-bit format's conversions, the
// writing of rows and the checks of a cache's descriptor.  Everything sits in an
// anonymous namespace: each .hip file is a translation unit of its own.  The
// layout is documented in include/vramc_kv.h.
#ifndef VRAMC_KV_DEVICE_H
#define VRAMC_KV_DEVICE_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/vramc_kv.h"

namespace {

constexpr int kMxBlock = 32;  // values to a scale byte
constexpr int64_t kMaxTokens = 1 << 29;  // that a row of the table has room for
constexpr int64_t kMaxThreads = UINT32_MAX;  // of a launch

template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// Two values of a byte of codes (the lower half first) times 2^(scale - 127).
template <typename T, int BYTE>
__device__ __forceinline__ uint32_t mx_pair(uint32_t codes, uint32_t scale) {
    const float unit = __uint_as_float(scale << 23);  // the conversion reads the exponent alone
    if constexpr (std::is_same_v<T, __bf16>)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, unit, BYTE));
    else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, unit, BYTE));
}
template <typename T>
__device__ __forceinline__ uint32_t mx_pair_at(uint32_t codes, uint32_t scale, int byte) {
    switch (byte) {  // constant after unrolling
        case 0: return mx_pair<T, 0>(codes, scale);
        case 1: return mx_pair<T, 1>(codes, scale);
        case 2: return mx_pair<T, 2>(codes, scale);
        default: return mx_pair<T, 3>(codes, scale);
    }
}

// The sum over a wave's lanes up to and with this one: within rows of 16 lanes,
// then each row's last lane into the rows behind it.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);   // row_shr:2
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);   // row_shr:4
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);   // row_shr:8
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
    return x;
}

constexpr int kPer = 8;  // values of a thread that copies rows

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

// The checks of every entry point.
inline int check_cache(const vramc_kv_cache* c) {
    if (!c || !c->k || !c->v || c->pages <= 0 || c->kv_heads <= 0) return RANS_EARG;
    switch (c->page_size) {
        case 16: case 32: case 64: case 128: case 256: break;
        default: return RANS_EUNSUPPORTED;
    }
    switch (c->head_dim) {
        case 64: case 96: case 128: case 192: case 256: break;
        default: return RANS_EUNSUPPORTED;
    }
    if (c->dtype != RANS_X_F32 && c->dtype != RANS_X_BF16 && c->dtype != RANS_X_F16)
        return RANS_EUNSUPPORTED;
    if (c->mx && c->dtype == RANS_X_F32) return RANS_EUNSUPPORTED;
    if (c->mx && (!c->k_scale || !c->v_scale)) return RANS_EARG;
    if (((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->mass | (uintptr_t)c->position) % 16) return RANS_EARG;
    if (!c->mass != !c->position) return RANS_EARG;
    return 0;
}

// Memory that a call reads or writes; no address or no bytes: none.
struct Span {
    const void* at;
    int64_t bytes;
};
inline bool overlap(Span a, Span b) {
    return a.at && b.at && a.bytes > 0 && b.bytes > 0 && (uintptr_t)a.at < (uintptr_t)b.at + b.bytes &&
           (uintptr_t)b.at < (uintptr_t)a.at + a.bytes;
}
template <size_t N, size_t M>
bool overlap(const Span (&a)[N], const Span (&b)[M]) {
    for (const Span& x : a)
        for (const Span& y : b)
            if (overlap(x, y)) return true;
    return false;
}

// Rows of `dim` values of `size` bytes each, x[t * token + h * head].
inline Span span_of(const void* x, int64_t token, int64_t head, int64_t tokens, int64_t heads, int64_t dim, int64_t size) {
    if (!x || tokens <= 0 || heads <= 0 || dim <= 0) return {};
    const int64_t far[] = {(tokens - 1) * token, (heads - 1) * head};
    int64_t first = 0, end = dim;
    for (const int64_t f : far) (f < 0 ? first : end) += f;
    return {static_cast<const char*>(x) + first * size, (end - first) * size};
}

// Pages of a cache's heads; more than these do not exist.
inline int64_t head_pages(const vramc_kv_cache& c) {
    const int64_t n = (int64_t)c.pages * c.kv_heads, most = INT64_MAX >> 20;
    return n < most ? n : most;
}

// The tensors of a cache.
struct CacheSpans {
    Span of[6];
};
inline CacheSpans spans_of(const vramc_kv_cache& c) {
    const int64_t tokens = head_pages(c) * c.page_size;
    const int64_t values = tokens * c.head_dim, size = c.dtype == RANS_X_F32 ? 4 : 2;
    const int64_t held = c.mx ? values / 2 : values * size, scales = c.mx ? values / 32 : 0;
    return {{{c.k, held}, {c.v, held}, {c.k_scale, scales}, {c.v_scale, scales}, {c.mass, 4 * tokens},
             {c.position, 4 * tokens}}};
}

}  // namespace

#endif  // VRAMC_KV_DEVICE_H
