// What the key-value cache's kernels share: the 4-bit format's conversions and
// the checks of a cache's descriptor.  Everything sits in an anonymous
// namespace: each .hip file is a translation unit of its own.  The layout is
// documented in include/vramc_kv.h.
#ifndef VRAMC_KV_DEVICE_H
#define VRAMC_KV_DEVICE_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/vramc_kv.h"

namespace {

constexpr int kMxBlock = 32;  // values to a scale byte
constexpr int64_t kMaxTokens = 1 << 30;  // that a row of the table has room for

template <typename T, int N>
using vec = T __attribute__((ext_vector_type(N)));

// 2^(s-127) of a scale byte, whose bits are a float's exponent: 0 is the
// subnormal 2^-127, 255 NaN.
__device__ __forceinline__ float mx_power(uint32_t s) {
    const uint32_t bits = s == 0 ? 0x00400000u : s == 255 ? 0x7fc00000u : s << 23;
    return __uint_as_float(bits);
}

// The value of a 4-bit code: 2^(e-1) * (1 + m/2), or m/2 where e is 0.
__device__ __forceinline__ float mx_value(uint32_t code) {
    const uint32_t e = code >> 1 & 3, m = code & 1;
    const float a = e ? __uint_as_float((e + 126) << 23 | m << 22) : 0.5f * (float)m;
    return code & 8 ? -a : a;
}

inline int size_of(int dtype) { return dtype == RANS_X_F32 ? 4 : 2; }

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
    if (((uintptr_t)c->k | (uintptr_t)c->v) % 16 || (!c->mass != !c->position)) return RANS_EARG;
    return 0;
}

}  // namespace

#endif  // VRAMC_KV_DEVICE_H
