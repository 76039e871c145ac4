// RMS norms of queries and keys for each head and their rotation by positions, in
// one pass, the keys and values into tensors or into the pages of a cache.
//
// Every value is read and written once, and HBM bounds it: 32768 tokens of 40 and 8
// heads of 128 columns, bf16, 159 us, 5.06 TB/s (a large copy reaches 4.8), 16001
// with their values into pages 98.7 us.  One token of 12 and 2 heads takes 3.3 us.
//
// A thread takes eight columns of a head, 16 bytes of a 16-bit type, a row of the
// workgroup's threads one head, so that the norm is a sum over at most 32 lanes.  The
// columns that its own rotate with are read again, from the caches, by the same
// thread: no exchange.  The next row's are under way while a row is turned (163 us
// without), and queries leave past the caches (168 us through them).
//
// A workgroup takes some tokens of one kind (queries, keys or values) with all
// their heads.  The angles are the same for all heads of a token: one thread makes
// each, to LDS.  position * turns is the angle in full turns, so that what it has
// of whole ones falls away exactly in 64 bits, and 32 hold the rest, for f32 rows with
// a first-order step for the bits beyond.
#include "kv_device.h"

#include "../../include/vramc_rotary.h"

namespace {

constexpr int kThreads = 256;
constexpr int kMostShift = 5;  // tokens of a workgroup, whose angles then take 8 KB of LDS at most

// Rows of one kind: `heads` of each token; how workgroups take them.
struct Kind {
    const void* x;
    int64_t token, head;     // strides
    const void* weight;
    void* out;
    int heads;
    bool wide;               // rows can be read 16 bytes at a time
    int shift;               // a workgroup has 2^shift tokens,
    int splits, passes;      // and takes `passes` of the steps of one of `splits`
    uint32_t blocks;
};

struct Rotate {
    Kind kind[3];            // queries, keys, values
    const double* turns;
    int pairs, dim, lanes;   // lanes: of a row, a power of two
    float amplitude, eps;
    bool weight_f32;
    const int32_t* positions;
    int tokens;
    // where keys and values go into a cache
    vramc_kv_cache c;
    int page_shift;
    const int64_t* slots;
};

// Eight values as they lie, rows aligned to 16 bytes where they are wide.
template <typename T>
__device__ __forceinline__ vec<T, kPer> load(const T* p, bool wide) {
    if (wide) return __builtin_bit_cast(vec<T, kPer>, *reinterpret_cast<const Lying<T>*>(p));
    vec<T, kPer> x;
#pragma unroll
    for (int j = 0; j < kPer; j++) x[j] = p[j];
    return x;
}

template <typename T>
__device__ __forceinline__ vec<float, kPer> floats(vec<T, kPer> x) {
    if constexpr (std::is_same_v<T, float>) return x;
    else return __builtin_convertvector(x, vec<float, kPer>);
}

// The sum over the lanes of a row, 8 to 32: within each half of 16 lanes by moves
// that mirror it, then over the halves.
__device__ __forceinline__ float row_sum(float x, int lanes) {
    const auto add = [&](auto control) {
        x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), control(), 0xf, 0xf, true));
    };
    add([] { return 0xb1; });   // quad_perm:[1,0,3,2]
    add([] { return 0x4e; });   // quad_perm:[2,3,0,1]
    add([] { return 0x141; });  // row_half_mirror
    if (lanes >= 16) add([] { return 0x140; });  // row_mirror
    if (lanes == 32) x += __shfl_xor(x, 16);
    return x;
}

enum Into { kTensor, kPlain, kMx };

template <typename T, bool INTERLEAVED, Into INTO>
__global__ void __launch_bounds__(kThreads) rotate_kernel(Rotate a) {
    extern __shared__ __attribute__((aligned(16))) float angles[];  // [token][cosines, sines][pairs]
    // this workgroup's kind, tokens and steps
    const int which = blockIdx.x < a.kind[0].blocks ? 0 : blockIdx.x - a.kind[0].blocks < a.kind[1].blocks ? 1 : 2;
    const Kind& k = a.kind[which];
    const uint32_t block = blockIdx.x - (which > 0 ? a.kind[0].blocks : 0) - (which > 1 ? a.kind[1].blocks : 0);
    const int tile = block / k.splits, part = block - tile * k.splits;
    const int first = tile << k.shift, tokens = min(a.tokens - first, 1 << k.shift);
    const int thread = threadIdx.y * a.lanes + threadIdx.x;
    if (which < 2) {
        for (int i = thread; i < tokens * a.pairs; i += kThreads) {
            const int t = i / a.pairs, j = i - t * a.pairs;
            const double turn = (double)a.positions[first + t] * a.turns[j];
            const double rest = turn - __builtin_rint(turn);
            float sine, cosine;
            sincospif(2.f * (float)rest, &sine, &cosine);
            if constexpr (std::is_same_v<T, float>) {  // what the rest's rounding left, no 16-bit type sees
                const float more = (float)(rest - (double)(float)rest) * 6.28318531f, before = cosine;
                cosine -= more * sine;
                sine += more * before;
            }
            angles[2 * t * a.pairs + j] = cosine * a.amplitude;
            angles[(2 * t + 1) * a.pairs + j] = sine * a.amplitude;
        }
        __syncthreads();
    }
    const int seg = threadIdx.x, column = kPer * seg, per_row = a.dim / kPer;
    const bool inside = seg < per_row, turned = inside && column < 2 * a.pairs;
    // the columns that these rotate with, the angles of both, and which way
    const bool second = !INTERLEAVED && column >= a.pairs;
    const int other = !turned ? column : second ? column - a.pairs : column + a.pairs;
    const int angle = INTERLEAVED ? column / 2 : second ? column - a.pairs : column;
    const bool norm = which < 2 && k.weight;
    vec<float, kPer> w = {}, w_other = {};
    if (norm && inside) {
        const auto take = [&](int at) {
            if (a.weight_f32) return load(static_cast<const float*>(k.weight) + at, true);
            return floats(load(static_cast<const T*>(k.weight) + at, true));
        };
        w = take(column);
        if constexpr (!INTERLEAVED) w_other = take(other);
    }
    const float share = 1.f / a.dim;
    const int rows = k.heads << k.shift, step = blockDim.y;
    int row = part * k.passes * step + threadIdx.y;
    // the row's token and head, and how far a step goes
    int t = row / k.heads, head = row - t * k.heads;
    const int t_step = step / k.heads, head_step = step - t_step * k.heads;
    const int stop = min(rows, row + k.passes * step);
    // a row's columns and those that they rotate with, and its place in the cache;
    // the next row's are under way while a row is turned
    vec<T, kPer> raw = {}, raw_other = {}, next = {}, next_other = {};
    int64_t at = -1, next_at = -1;
    const auto fetch = [&](int t, int head) {
        if (t >= tokens) return;
        if (inside) {
            const T* in = static_cast<const T*>(k.x) + (first + t) * k.token + head * k.head;
            next = load(in + column, k.wide);
            if constexpr (!INTERLEAVED)
                if (which < 2) next_other = load(in + other, k.wide);
        }
        if (INTO != kTensor && which > 0) {
            const int64_t slot = a.slots[first + t];
            next_at = slot >= 0 && slot < (int64_t)a.c.pages << a.page_shift
                          ? (((slot >> a.page_shift) * a.c.kv_heads + head) << a.page_shift) + (slot & (a.c.page_size - 1))
                          : -1;
        }
    };
    if (row < stop) fetch(t, head);
    while (row < stop) {
        const int this_t = t, this_head = head;
        raw = next, raw_other = next_other, at = next_at;
        row += step;
        t += t_step, head += head_step;
        if (head >= k.heads) head -= k.heads, t++;
        if (row < stop) fetch(t, head);
        if (this_t < tokens) {  // lanes beyond the row take part in its sum
            vec<T, kPer> y;
            if (which == 2) {
                y = raw;
            } else {
                vec<float, kPer> x = floats(raw), z;
                float scale = 1.f;
                if (norm) {
                    float squares = 0.f;
#pragma unroll
                    for (int j = 0; j < kPer; j++) squares += x[j] * x[j];
                    scale = rsqrtf(row_sum(squares, a.lanes) * share + a.eps);
                    x *= w;
                }
                if (turned) {
                    const float* cs = angles + 2 * this_t * a.pairs + angle;
                    if constexpr (INTERLEAVED) {
#pragma unroll
                        for (int j = 0; j < kPer; j += 2) {
                            const float cosine = cs[j / 2], sine = cs[a.pairs + j / 2];
                            z[j] = x[j] * cosine - x[j + 1] * sine;
                            z[j + 1] = x[j + 1] * cosine + x[j] * sine;
                        }
                    } else {
                        vec<float, kPer> x_other = floats(raw_other);
                        if (norm) x_other *= w_other;
#pragma unroll
                        for (int j = 0; j < kPer; j++) {
                            const float sine = cs[a.pairs + j];
                            z[j] = x[j] * cs[j] + x_other[j] * (second ? sine : -sine);
                        }
                    }
                } else {
                    z = x;
                }
                z *= scale;
                if constexpr (std::is_same_v<T, float>) y = z;
                else y = __builtin_convertvector(z, vec<T, kPer>);
            }
            if (!inside) {
            } else if (INTO == kTensor || which == 0) {
                auto* out = static_cast<Lying<T>*>(k.out) + ((int64_t)(first + this_t) * k.heads + this_head) * per_row + seg;
                const auto part = __builtin_bit_cast(Lying<T>, y);
#pragma unroll
                for (size_t j = 0; j < sizeof(T) / 2; j++) __builtin_nontemporal_store(part.part[j], &out->part[j]);
            } else if constexpr (INTO != kTensor) {
                if (at >= 0) {  // a block's threads share it
                    store<T, INTO == kMx>(y, which == 1 ? a.c.k : a.c.v, which == 1 ? a.c.k_scale : a.c.v_scale, at,
                                          per_row, seg);
                    if (which == 1 && a.c.mass && seg == 0) {
                        a.c.mass[at] = 0.f;
                        a.c.position[at] = a.positions[first + this_t];
                    }
                }
            }
        }
    }
}

int check(const vramc_rotary* r, const vramc_rotary_rows* x) {
    if (!r || !x || !r->turns) return RANS_EARG;
    switch (r->head_dim) {
        case 64: case 96: case 128: case 192: case 256: break;
        default: return RANS_EUNSUPPORTED;
    }
    if (r->pairs <= 0 || r->pairs % 8 || 2 * r->pairs > r->head_dim) return RANS_EUNSUPPORTED;
    if (x->dtype != RANS_X_F32 && x->dtype != RANS_X_BF16 && x->dtype != RANS_X_F16) return RANS_EUNSUPPORTED;
    const bool weights = x->q_weight || x->k_weight;
    if (weights && x->weight_dtype != RANS_X_F32 && x->weight_dtype != x->dtype) return RANS_EUNSUPPORTED;
    if (x->q_heads < 0 || x->k_heads < 0 || !(x->eps >= 0) || x->tokens < 0) return RANS_EARG;
    if (x->q_token < 0 || x->q_head < 0 || x->k_token < 0 || x->k_head < 0) return RANS_EARG;
    // rows are counted in 32 bits, and a launch has fewer than 2^32 threads
    const int64_t most = (int64_t)(x->q_heads > x->k_heads ? x->q_heads : x->k_heads);
    if (x->tokens > (1 << 26) || most > (1 << 16) || x->tokens * most > (1 << 26)) return RANS_EARG;
    if (x->tokens && (!x->positions || (x->q_heads && !x->q) || (x->k_heads && !x->k))) return RANS_EARG;
    if (((uintptr_t)x->q_weight | (uintptr_t)x->k_weight) % 16) return RANS_EARG;
    return 0;
}

int64_t size_of(int dtype) { return dtype == RANS_X_F32 ? 4 : 2; }

// What both calls read.
struct RowsSpans {
    Span of[6];
};
RowsSpans spans_of(const vramc_rotary& r, const vramc_rotary_rows& x) {
    const int64_t dim = r.head_dim, size = size_of(x.dtype), weight = dim * size_of(x.weight_dtype);
    return {{span_of(x.q, x.q_token, x.q_head, x.tokens, x.q_heads, dim, size),
             span_of(x.k, x.k_token, x.k_head, x.tokens, x.k_heads, dim, size),
             {x.q_weight, weight}, {x.k_weight, weight}, {x.positions, x.tokens * 4}, {r.turns, r.pairs * (int64_t)8}}};
}

template <typename T>
Kind kind_of(const void* x, int64_t token, int64_t head, int heads, const void* weight, void* out, int64_t tokens,
             int lanes) {
    Kind k{x, token, head, weight, out, heads, false, 0, 1, 0, 0};
    if (!heads || !tokens) return k;
    constexpr int64_t size = sizeof(T);
    k.wide = ((uintptr_t)x | (uintptr_t)(token * size) | (uintptr_t)(head * size)) % 16 == 0;
    const int step = kThreads / lanes;
    // Tokens of a workgroup: more share less of the angles and end later.  40 and 8 heads
    // of 128 columns, bf16: 512 tokens 6.7 us by two and 6.4 by one with its heads dealt
    // to several workgroups, 1000 8.4 and 11.0; 2048 12.0 by two and 12.7 by four, 4096
    // 20.5 and 18.6, 32768 175 and 159 (by eight 161).
    k.shift = tokens >= 4096 ? 2 : tokens >= 512 ? 1 : 0;
    // and of many tokens so many that few heads leave no threads without a row (16384
    // tokens of one head of 64 columns 6.6 us against 13.3; 1000 are better spread)
    if (tokens >= 4096)
        while (heads << k.shift < step && k.shift < kMostShift) k.shift++;
    const int steps = ((heads << k.shift) + step - 1) / step;
    k.splits = k.shift ? 1 : steps;
    k.passes = k.shift ? steps : 1;
    k.blocks = (uint32_t)((tokens + (1 << k.shift) - 1) >> k.shift) * (uint32_t)k.splits;
    return k;
}

template <typename T, Into INTO>
int launch(const vramc_rotary& r, const vramc_rotary_rows& x, const vramc_kv_cache* c, const void* v, int64_t v_token,
           int64_t v_head, const int64_t* slots, void* q_out, void* k_out, hipStream_t stream) {
    const int lanes = r.head_dim <= 64 ? 8 : r.head_dim <= 128 ? 16 : 32;
    constexpr bool pages = INTO != kTensor;
    Rotate a{};
    a.kind[0] = kind_of<T>(x.q, x.q_token, x.q_head, x.q_heads, x.q_weight, q_out, x.tokens, lanes);
    a.kind[1] = kind_of<T>(x.k, x.k_token, x.k_head, x.k_heads, x.k_weight, k_out, x.tokens, lanes);
    a.kind[2] = kind_of<T>(v, v_token, v_head, pages ? x.k_heads : 0, nullptr, nullptr, x.tokens, lanes);
    a.turns = r.turns, a.pairs = r.pairs, a.dim = r.head_dim, a.lanes = lanes;
    a.amplitude = r.amplitude, a.eps = x.eps, a.weight_f32 = x.weight_dtype == RANS_X_F32;
    a.positions = x.positions, a.tokens = (int)x.tokens;
    if (pages) a.c = *c, a.page_shift = __builtin_ctz(c->page_size), a.slots = slots;
    const int64_t blocks = (int64_t)a.kind[0].blocks + a.kind[1].blocks + a.kind[2].blocks;
    if (blocks == 0) return 0;
    if (blocks > kMaxThreads / kThreads) return RANS_EARG;
    const int shift = a.kind[0].shift > a.kind[1].shift ? a.kind[0].shift : a.kind[1].shift;
    const size_t lds = (size_t)(8 * r.pairs) << shift;
    const dim3 grid((unsigned)blocks), block((unsigned)lanes, (unsigned)(kThreads / lanes));
    if (r.interleaved) hipLaunchKernelGGL((rotate_kernel<T, true, INTO>), grid, block, lds, stream, a);
    else hipLaunchKernelGGL((rotate_kernel<T, false, INTO>), grid, block, lds, stream, a);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" int vramc_rotary_apply(const vramc_rotary* r, const vramc_rotary_rows* x, void* q_out, void* k_out,
                                  hipStream_t stream) {
    if (const int rc = check(r, x)) return rc;
    if (x->tokens == 0) return 0;
    if ((x->q_heads && !q_out) || (x->k_heads && !k_out) || ((uintptr_t)q_out | (uintptr_t)k_out) % 16) return RANS_EARG;
    const int64_t value = size_of(x->dtype) * r->head_dim;
    const Span out[] = {{q_out, x->tokens * x->q_heads * value}, {k_out, x->tokens * x->k_heads * value}};
    if (overlap(out[0], out[1]) || overlap(out, spans_of(*r, *x).of)) return RANS_EARG;
    const auto go = [&](auto fn) { return fn(*r, *x, nullptr, nullptr, 0, 0, nullptr, q_out, k_out, stream); };
    if (x->dtype == RANS_X_F32) return go(launch<float, kTensor>);
    return x->dtype == RANS_X_BF16 ? go(launch<__bf16, kTensor>) : go(launch<_Float16, kTensor>);
}

extern "C" int vramc_rotary_append(const vramc_rotary* r, const vramc_rotary_rows* x, const vramc_kv_cache* c,
                                   const void* v, int64_t v_token, int64_t v_head, const int64_t* slots, void* q_out,
                                   hipStream_t stream) {
    if (const int rc = check(r, x)) return rc;
    if (const int rc = check_cache(c)) return rc;
    if (c->head_dim != r->head_dim || c->dtype != x->dtype || c->kv_heads != x->k_heads || v_token < 0 || v_head < 0)
        return RANS_EARG;
    if (x->tokens == 0) return 0;
    if (!v || !slots || (x->q_heads && !q_out) || (uintptr_t)q_out % 16) return RANS_EARG;
    const Span out[] = {{q_out, x->tokens * x->q_heads * size_of(x->dtype) * r->head_dim}};
    const Span more[] = {span_of(v, v_token, v_head, x->tokens, x->k_heads, r->head_dim, size_of(x->dtype)),
                         {slots, x->tokens * 8}};
    const auto read = spans_of(*r, *x);
    const auto pages = spans_of(*c);
    if (overlap(out, read.of) || overlap(out, more) || overlap(out, pages.of) || overlap(pages.of, read.of) ||
        overlap(pages.of, more))
        return RANS_EARG;
    const auto go = [&](auto fn) { return fn(*r, *x, c, v, v_token, v_head, slots, q_out, nullptr, stream); };
    if (x->dtype == RANS_X_F32) return go(launch<float, kPlain>);
    if (x->dtype == RANS_X_BF16) return c->mx ? go(launch<__bf16, kMx>) : go(launch<__bf16, kPlain>);
    return c->mx ? go(launch<_Float16, kMx>) : go(launch<_Float16, kPlain>);
}
