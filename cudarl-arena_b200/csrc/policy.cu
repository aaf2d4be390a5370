// policy.cu -- log probabilities of the actions taken, entropy and most probable alternatives of rows of logits, and the gradient of the logits.
//
// Row x, legal actions L, scale = 1 / temperature, m = max x.  In base 2, with c = scale log2(e):
//   y = x c - m c <= 0,   S = sum 2^y,   log2 p = y - log2 S,   H = ln 2 (log2 S - (sum y 2^y) / S)      (both terms >= 0: nothing cancels)
//   dx_j = scale (gl ([j = taken] - p_j) - gH p_j (ln p_j + H))
// What a row of more than 128 actions leaves for its gradient: {m, log2 S, H}.
//
// What bounds it (B200, times of the kernels alone): long rows the memory and, a step behind, the exponentials (16 a cycle and SM): 4096 x 131072 bf16, 1.07 GB, 178 us =
// 6.0 TB/s without alternatives, 207 us with 5; its gradient, 2047 x 65537, 0.54 GB, 88 us = 6.1 TB/s.  Short rows the instructions that are made once a row:
// 4,194,304 x 4 fp32 26.6 us forward (2.5 TB/s of logits, 4.4 with the actions and the results), gradient 37 us.
//
// y is one fused multiply-add with m c rounded once: an error of m c multiplies all 2^y of the row alike and leaves p as it is, so long as every
// use takes the same m c.  Minus infinity, masked places and whatever is below FLOOR count as FLOOR (2^y is 0 there all the same), so y 2^y needs no
// test.  Rows with |m c| of 2^23 and more, where the error would be whole powers of two, are gone through a second time with exact differences.
#include "caller_arrays.cuh"
#include <cooperative_groups.h>

namespace {
using namespace cudarl;
namespace cg = cooperative_groups;

constexpr float NONE = -INFINITY, FLOOR = -1e20f, ABOVE_FLOOR = -9e19f, LARGE = 1e19f, LIMIT = 8388608.0f;
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.693147180559945309417f;
constexpr unsigned ALL = 0xFFFFFFFFu;

struct Rows {
    const void* logits;
    const unsigned char* legal;
    const int* taken;
    long long rows, stride, legal_stride;
    int actions;
    float scale;                       // 1 / temperature
};
struct Outputs {
    float* logprob; float* entropy; float4* stats; int* top_actions; float* top_logprobs;
    int top;
};

// ------------------------------------------------------------------------------------------------------------------ arithmetic
__device__ __forceinline__ float exp2_fast(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float max3(float a, float b, float c) { float r; asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
__device__ __forceinline__ float sum2(Two v) { float a, b; apart(v, a, b); return a + b; }

// Larger for the larger logit, of equal ones for the lower action; 0 for none.
__device__ __forceinline__ unsigned long long order_key(float x, unsigned action) {
    const unsigned b = __float_as_uint(x + 0.0f);                            // -0 counts as 0
    return ((unsigned long long)((b & 0x80000000u) ? ~b : b | 0x80000000u) << 32) | (0xFFFFFFFFu - action);
}
__device__ __forceinline__ float key_value(unsigned long long key) {
    const unsigned b = (unsigned)(key >> 32);
    return __uint_as_float((b & 0x80000000u) ? b & 0x7FFFFFFFu : ~b);
}
// The same for a value of 16 bits and an action below 2^16, in 32 bits.
template <int TYPE> __device__ __forceinline__ unsigned order_key16(float x, unsigned action) {
    x += 0.0f;
    const unsigned b = TYPE == CUDARL_BF16 ? __float_as_uint(x) >> 16 : (unsigned)__half_as_ushort(__float2half_rn(x));
    return ((b & 0x8000u) ? ~b & 0xFFFFu : b | 0x8000u) << 16 | (0xFFFFu - action);
}
template <int TYPE> __device__ __forceinline__ float key16_value(unsigned key) {
    const unsigned b = (key & 0x80000000u) ? key >> 16 & 0x7FFFu : ~(key >> 16) & 0xFFFFu;
    return TYPE == CUDARL_BF16 ? __uint_as_float(b << 16) : __half2float(__ushort_as_half((unsigned short)b));
}
__device__ __forceinline__ int key_action(unsigned long long key) { return (int)(0xFFFFFFFFu - (unsigned)key); }

// A part of a row: its maximum, and the sums with the maximum's m c taken off -- or -LIMIT where that is more: a part so low (a masked one, or an empty one)
// leaves sums of nothing then, not of rounding errors.
struct Part { float m, s, t; };
__device__ __forceinline__ float base_of(float m, float c) { return fmaxf(m * c, -LIMIT); }
__device__ __forceinline__ bool is_usual(float m, float c) { return fabsf(m * c) < LIMIT; }
__device__ __forceinline__ void rebase(Part& p, float m, float c) {          // the same sums for another (higher) maximum: y - by, 2^-by as much
    const float by = base_of(m, c) - base_of(p.m, c), r = exp2_fast(-by);
    p.t = r * (p.t - by * p.s);
    p.s *= r;
    p.m = m;
}
__device__ __forceinline__ void take_one(Part& p, float x, float c) {
    if (x > p.m) rebase(p, x, c);
    const float y = fmaf(max_nan(x, FLOOR), c, -base_of(p.m, c)), e = exp2_fast(y);
    p.s += e;
    p.t = fmaf(y, e, p.t);
}
// What is known of a whole row.
struct Known {
    float m, log2_s, h;
    bool nothing, bad;                                                       // no action has any probability; a NaN or plus infinity is among them
    __device__ __forceinline__ Known(const Part& p) {
        nothing = p.s == 0.0f; bad = !(p.s == p.s);
        m = p.m; log2_s = __log2f(p.s); h = nothing ? 0.0f : max_nan(LN2 * (log2_s - __fdividef(p.t, p.s)), 0.0f);      // (s is 1 or more: both are good to some 2^-22)
    }
    // Log probability of an action with this logit.
    __device__ __forceinline__ float logprob(float x, const Rows& p) const {
        if (bad) return log2_s;
        if (x == NONE || nothing) return NONE;
        const float c = p.scale * LOG2E;
        if (!(fabsf(x) < LARGE && is_usual(m, c))) return (x - m) * p.scale - LN2 * log2_s;
        return fminf(LN2 * (fmaf(x, c, -(m * c)) - log2_s), 0.0f);
    }
    __device__ __forceinline__ void write(const Outputs& o, long long r) const {
        if (o.entropy) o.entropy[r] = h;
        if (o.stats) o.stats[r] = make_float4(m, log2_s, h, 0.0f);
    }
};

// ------------------------------------------------------------------------------------------------------------------ loads of 16 bytes
template <int TYPE> struct Chunk;
template <> struct Chunk<CUDARL_F32> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void values(const uint4& v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 fill() { return make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u); }                // minus infinities
    static __device__ __forceinline__ void floored(const uint4& v, float (&x)[4]) {
        values(v, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = max_nan(x[i], FLOOR);
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[4]) { return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])); }
};
template <> struct Chunk<CUDARL_BF16> {
    static constexpr int N = 8;
    static constexpr unsigned FLOOR2 = 0xE0ADE0ADu;                          // FLOOR, rounded to bf16, twice
    static __device__ __forceinline__ void pair(unsigned v, float& a, float& b) { a = __uint_as_float(v << 16); b = __uint_as_float(v & 0xFFFF0000u); }
    static __device__ __forceinline__ void values(const uint4& v, float (&x)[8]) { pair(v.x, x[0], x[1]); pair(v.y, x[2], x[3]); pair(v.z, x[4], x[5]); pair(v.w, x[6], x[7]); }
    static __device__ __forceinline__ uint4 fill() { return make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u); }
    static __device__ __forceinline__ unsigned up(unsigned v) { unsigned r; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(FLOOR2)); return r; }
    static __device__ __forceinline__ void floored(const uint4& v, float (&x)[8]) { values(make_uint4(up(v.x), up(v.y), up(v.z), up(v.w)), x); }
    static __device__ __forceinline__ unsigned two16(float a, float b) { const __nv_bfloat162 v = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const unsigned*>(&v); }
    static __device__ __forceinline__ uint4 pack(const float (&x)[8]) { return make_uint4(two16(x[0], x[1]), two16(x[2], x[3]), two16(x[4], x[5]), two16(x[6], x[7])); }
};
template <> struct Chunk<CUDARL_F16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void pair(unsigned v, float& a, float& b) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v)); a = f.x; b = f.y; }
    static __device__ __forceinline__ void values(const uint4& v, float (&x)[8]) { pair(v.x, x[0], x[1]); pair(v.y, x[2], x[3]); pair(v.z, x[4], x[5]); pair(v.w, x[6], x[7]); }
    static __device__ __forceinline__ uint4 fill() { return make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u); }
    static __device__ __forceinline__ void floored(const uint4& v, float (&x)[8]) {
        values(v, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = max_nan(x[i], FLOOR);
    }
    static __device__ __forceinline__ unsigned two16(float a, float b) { const __half2 v = __floats2half2_rn(a, b); return *reinterpret_cast<const unsigned*>(&v); }
    static __device__ __forceinline__ uint4 pack(const float (&x)[8]) { return make_uint4(two16(x[0], x[1]), two16(x[2], x[3]), two16(x[4], x[5]), two16(x[6], x[7])); }
};

// The same from an address that is not aligned.
__device__ __forceinline__ uint4 gather_chunk(const float* at) {
    return make_uint4(__float_as_uint(at[0]), __float_as_uint(at[1]), __float_as_uint(at[2]), __float_as_uint(at[3]));
}
template <class Half> __device__ __forceinline__ uint4 gather_chunk(const Half* at) {
    static_assert(sizeof(Half) == 2, "");
    const unsigned short* v = reinterpret_cast<const unsigned short*>(at);
    return make_uint4(v[0] | (unsigned)v[1] << 16, v[2] | (unsigned)v[3] << 16, v[4] | (unsigned)v[5] << 16, v[6] | (unsigned)v[7] << 16);
}

// The mask bytes of N actions from `j` on, in words.  Inside a row: the aligned words that hold them, shifted; at its ends one by one.
template <int N>
__device__ __forceinline__ void mask_words(const unsigned char* legal, int j, int actions, unsigned (&w)[N / 4]) {
    const unsigned char* at = legal + j;
    const unsigned off = (unsigned)reinterpret_cast<uintptr_t>(at) & 3u;
    if (off == 0u) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) w[i] = __ldg(reinterpret_cast<const unsigned*>(at) + i);
    } else if (j >= 3 && j + N + 3 <= actions) {
        const unsigned* a = reinterpret_cast<const unsigned*>(at - off);
        unsigned before = __ldg(a);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) { const unsigned next = __ldg(a + i + 1); w[i] = __funnelshift_r(before, next, 8u * off); before = next; }
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) w[i] = __ldg(at + 4 * i) | __ldg(at + 4 * i + 1) << 8 | __ldg(at + 4 * i + 2) << 16 | (unsigned)__ldg(at + 4 * i + 3) << 24;
    }
}
template <int N> __device__ __forceinline__ bool is_legal(const unsigned (&w)[N / 4], int i) { return (w[i / 4] & (0xFFu << (8 * (i % 4)))) != 0u; }

// One row: its values one by one, and its 16-byte chunks -- the first begins at the first aligned address; the values before it and behind the last, fewer
// than two chunks of them, are the row's ends.
template <int TYPE>
struct Row {
    using O = Of<TYPE>;
    static constexpr int N = Chunk<TYPE>::N;
    const typename O::T* x; const unsigned char* legal;
    int actions, head, chunks, ends;
    __device__ __forceinline__ Row(const Rows& p, long long r) {
        x = static_cast<const typename O::T*>(p.logits) + r * p.stride;
        legal = p.legal ? p.legal + r * p.legal_stride : nullptr;
        actions = p.actions;
        head = min((int)((16u - ((unsigned)reinterpret_cast<uintptr_t>(x) & 15u)) & 15u) / (int)sizeof(typename O::T), actions);
        chunks = (actions - head) / N;
        ends = actions - chunks * N;
    }
    __device__ __forceinline__ void move_to(const Rows& p, long long r) {    // to another row that lies as this one does to 16 bytes
        x = static_cast<const typename O::T*>(p.logits) + r * p.stride;
        if (legal) legal = p.legal + r * p.legal_stride;
    }
    __device__ __forceinline__ float at(int j) const { return legal && !__ldg(legal + j) ? NONE : O::get(x[j]); }
    __device__ __forceinline__ int end(int i) const { return i < head ? i : chunks * N + i; }       // the action of the i-th of the ends
    __device__ __forceinline__ uint4 chunk(int k) const { return __ldg(reinterpret_cast<const uint4*>(x + head) + k); }
};

// ------------------------------------------------------------------------------------------------------------------ order of the best
// 32 keys, one a lane, into falling order (bitonic).
__device__ __forceinline__ unsigned long long swap_with(unsigned long long key, unsigned lane, unsigned by, bool falling) {
    const unsigned long long other = __shfl_xor_sync(ALL, key, by);
    const bool keep_larger = ((lane & by) == 0u) == falling;
    return (key > other) == keep_larger ? key : other;
}
__device__ __forceinline__ unsigned long long sorted32(unsigned long long key, unsigned lane) {
#pragma unroll
    for (unsigned size = 2; size <= 32; size *= 2)
#pragma unroll
        for (unsigned by = size / 2; by; by /= 2) key = swap_with(key, lane, by, (lane & size) == 0u || size == 32u);
    return key;
}
// The 32 largest of two falling lists, falling.
__device__ __forceinline__ unsigned long long merged32(unsigned long long a, unsigned long long b, unsigned lane) {
    b = __shfl_sync(ALL, b, 31u - lane);
    a = a > b ? a : b;
#pragma unroll
    for (unsigned by = 16; by; by /= 2) a = swap_with(a, lane, by, true);
    return a;
}
// Takes 32 more keys (0 = none) into a falling list of which the first `top` count.
__device__ __forceinline__ void take32(unsigned long long& list, unsigned long long key, unsigned lane, int top) {
    const unsigned long long least = __shfl_sync(ALL, list, top - 1);
    if (__any_sync(ALL, key > least)) list = merged32(list, sorted32(key, lane), lane);
}

__device__ __forceinline__ void write_top(const Outputs& o, const Rows& p, const Known& known, long long r, int place, unsigned long long key) {
    o.top_actions[r * o.top + place] = key ? key_action(key) : -1;
    o.top_logprobs[r * o.top + place] = known.bad ? known.log2_s : key ? known.logprob(key_value(key), p) : NONE;
}

// ------------------------------------------------------------------------------------------------------------------ short rows
// G lanes a row, E values a lane in registers: up to G E actions (100 of them, 500,000 rows of bf16: 61 us, gradient 90; as a warp a row 109 and 180; from 129 on the
// two are alike without alternatives and 16 lanes the slower with 20 of them: 883 against 586 us for 500,000 x 256 fp32).  WIDE: a lane has neighbouring values and moves them at once, which takes rows that are aligned
// to that; else neighbouring lanes have neighbouring values, so that what a warp reads or writes at a time lies together.
template <int G, int E, bool WIDE> __device__ __forceinline__ int short_action(int lane, int i) { return WIDE ? lane * E + i : lane + G * i; }

template <int TYPE, int G, int E, bool WIDE>
__device__ __forceinline__ void load_short(const Rows& p, long long r, int lane, float (&x)[E]) {
    using O = Of<TYPE>;
    const auto* at = static_cast<const typename O::T*>(p.logits) + r * p.stride;
    constexpr int BYTES = E * (int)sizeof(typename O::T);
    if (WIDE && lane * E + E <= p.actions) {
        if constexpr (BYTES == 8 && TYPE != CUDARL_F32) {
            const uint2 v = *reinterpret_cast<const uint2*>(at + lane * E);
            Chunk<TYPE>::pair(v.x, x[0], x[1]); Chunk<TYPE>::pair(v.y, x[2], x[3]);
        } else if constexpr (BYTES >= 16) {
#pragma unroll
            for (int k = 0; k < BYTES / 16; ++k) {
                float part[Chunk<TYPE>::N];
                Chunk<TYPE>::values(reinterpret_cast<const uint4*>(at + lane * E)[k], part);
#pragma unroll
                for (int i = 0; i < Chunk<TYPE>::N; ++i) x[k * Chunk<TYPE>::N + i] = part[i];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) { const int j = short_action<G, E, WIDE>(lane, i); x[i] = j < p.actions ? O::get(at[j]) : NONE; }
    }
    if (p.legal) {
        const unsigned char* legal = p.legal + r * p.legal_stride;
#pragma unroll
        for (int i = 0; i < E; ++i) { const int j = short_action<G, E, WIDE>(lane, i); x[i] = j < p.actions && __ldg(legal + j) ? x[i] : NONE; }
    }
}

// y and 2^y of the lane's values, and the row's part in all its lanes.  `exact`: the row is beyond the limit.
template <int G, int E>
__device__ __forceinline__ Part sum_short(const float (&x)[E], float scale, float (&y)[E], float (&e)[E], bool& exact) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < E; ++i) m = fmaxf(m, x[i]);
#pragma unroll
    for (int by = 1; by < G; by *= 2) m = fmaxf(m, __shfl_xor_sync(ALL, m, by));
    const float c = scale * LOG2E, mc = m * c;
    exact = !is_usual(m, c);
    const Two c2 = two(c, c), mc2 = two(-mc, -mc);
#pragma unroll
    for (int i = 0; i < E; i += 2) apart(fma2(two(max_nan(x[i], FLOOR), max_nan(x[i + 1], FLOOR)), c2, mc2), y[i], y[i + 1]);
    if (__any_sync(ALL, exact)) {
        const float from = m == NONE ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < E; ++i) y[i] = exact ? max_nan((x[i] - from) * scale * LOG2E, FLOOR) : y[i];
    }
    Two s2 = two(0.0f, 0.0f), t2 = s2;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
        e[i] = exp2_fast(y[i]); e[i + 1] = exp2_fast(y[i + 1]);
        s2 = add2(s2, two(e[i], e[i + 1]));
        t2 = fma2(two(y[i], y[i + 1]), two(e[i], e[i + 1]), t2);
    }
    Part part{m, sum2(s2), sum2(t2)};
#pragma unroll
    for (int by = 1; by < G; by *= 2) { part.s += __shfl_xor_sync(ALL, part.s, by); part.t += __shfl_xor_sync(ALL, part.t, by); }
    return part;
}

template <int TYPE, int G, int E, bool WIDE, bool TOP>
__global__ void __launch_bounds__(256) k_short(Rows p, Outputs o) {
    const int lane = (int)threadIdx.x % G;
    const long long step = (long long)gridDim.x * (256 / G);
    // (the loop is the same for all lanes of a warp: rows behind the last are computed from the last and not written)
    for (long long first = (long long)blockIdx.x * (256 / G); first < p.rows; first += step) {
        const long long mine = first + (int)threadIdx.x / G, r = mine < p.rows ? mine : p.rows - 1;
        const bool write = mine < p.rows;
        float x[E], y[E], e[E];
        load_short<TYPE, G, E, WIDE>(p, r, lane, x);
        const int a = p.taken ? __ldg(p.taken + r) : -1;
        bool exact;
        const Known known(sum_short<G, E>(x, p.scale, y, e, exact));
        const bool rare = exact || known.bad;
        const float c = p.scale * LOG2E, base = -(known.m * c);
        auto logprob = [&](float v) { return rare || v < -LARGE ? known.logprob(v, p) : fminf(LN2 * (fmaf(v, c, base) - known.log2_s), 0.0f); };
        if (write && lane == 0) {
            if (o.entropy) o.entropy[r] = known.h;
            if (o.logprob) {
                float lp = known.bad ? known.log2_s : 0.0f;
                if constexpr (G == 1) {                                      // the lane has it
                    float xa = x[0];
#pragma unroll
                    for (int i = 1; i < E; ++i) xa = a == i ? x[i] : xa;
                    if ((unsigned)a < (unsigned)p.actions) lp = logprob(xa);
                } else if ((unsigned)a < (unsigned)p.actions)
                    lp = logprob(p.legal && !__ldg(p.legal + r * p.legal_stride + a) ? NONE : Of<TYPE>::get(static_cast<const typename Of<TYPE>::T*>(p.logits)[r * p.stride + a]));
                o.logprob[r] = lp;
            }
        }
        if constexpr (TOP) {
            // the largest of the row's remaining values, of equal ones the lowest action, `top` times
            if constexpr (TYPE != CUDARL_F32) {                              // 16 bits of value and 16 of action: one integer
                unsigned key[E];
#pragma unroll
                for (int i = 0; i < E; ++i) key[i] = x[i] > NONE && !known.bad ? order_key16<TYPE>(x[i], (unsigned)short_action<G, E, WIDE>(lane, i)) : 0u;
                int* const top_actions = o.top_actions + r * o.top;
                float* const top_logprobs = o.top_logprobs + r * o.top;
                for (int k = 0; k < o.top; ++k) {
                    unsigned best = key[0];
#pragma unroll
                    for (int i = 1; i < E; ++i) best = max(best, key[i]);
#pragma unroll
                    for (int by = 1; by < G; by *= 2) best = max(best, __shfl_xor_sync(ALL, best, by));
#pragma unroll
                    for (int i = 0; i < E; ++i) key[i] = key[i] == best ? 0u : key[i];
                    if (write && lane == 0) {
                        top_actions[k] = best ? (int)(0xFFFFu - (best & 0xFFFFu)) : -1;
                        top_logprobs[k] = best ? logprob(key16_value<TYPE>(best)) : known.bad ? known.log2_s : NONE;
                    }
                }
            } else {
                if (known.bad) {
#pragma unroll
                    for (int i = 0; i < E; ++i) x[i] = NONE;
                }
                int* const top_actions = o.top_actions + r * o.top;
                float* const top_logprobs = o.top_logprobs + r * o.top;
                for (int k = 0; k < o.top; ++k) {
                    float high = x[0];
#pragma unroll
                    for (int i = 1; i < E; ++i) high = fmaxf(high, x[i]);
#pragma unroll
                    for (int by = 1; by < G; by *= 2) high = fmaxf(high, __shfl_xor_sync(ALL, high, by));
                    int at = 0x7FFFFFFF;
#pragma unroll
                    for (int i = E - 1; i >= 0; --i) at = x[i] == high ? short_action<G, E, WIDE>(lane, i) : at;
#pragma unroll
                    for (int by = 1; by < G; by *= 2) at = min(at, __shfl_xor_sync(ALL, at, by));
                    const bool there = high > NONE;
#pragma unroll
                    for (int i = 0; i < E; ++i) x[i] = there && short_action<G, E, WIDE>(lane, i) == at ? NONE : x[i];
                    if (write && lane == 0) {
                        top_actions[k] = there ? at : -1;
                        top_logprobs[k] = there ? logprob(high) : known.bad ? known.log2_s : NONE;
                    }
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------ parts of warps
__device__ __forceinline__ float warp_max(float v) { float r; asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float warp_min(float v) { float r; asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v)); return r; }
// Has the bytes from `at` to `end` on their way to L2, a sector a thread at a time.
__device__ __forceinline__ void fetch_ahead(const void* at, const void* end, int t, int threads) {
    for (const char* a = static_cast<const char*>(at) + t * 32; a < static_cast<const char*>(end); a += threads * 32) asm volatile("prefetch.global.L2 [%0];" :: "l"(a));
}
// The 32 lanes' parts as one, in every lane.
__device__ __forceinline__ void join_lanes(Part& p, float c, int lanes = 32) {
    rebase(p, warp_max(p.m), c);
    for (int by = lanes / 2; by; by /= 2) { p.s += __shfl_xor_sync(ALL, p.s, by); p.t += __shfl_xor_sync(ALL, p.t, by); }
}
// The `rank`-th largest of the lanes' values (1 .. 32).
__device__ __forceinline__ float warp_ranked(float v, int rank) {
    while (true) {
        const float high = warp_max(v);
        rank -= __popc(__ballot_sync(ALL, v == high));
        if (rank <= 0 || high == NONE) return high;
        v = v == high ? NONE : v;
    }
}
// A whole row by the threads of a team a second time, with exact differences: lane- and warp-wise parts of it (see below for where it is needed).
template <int AT_ONCE, int TYPE, class F> __device__ __forceinline__ void each_chunk(const Row<TYPE>& row, int t, int threads, F f) {
    constexpr int N = Chunk<TYPE>::N;
#pragma unroll AT_ONCE
    for (int k = t; k < row.chunks; k += threads) {
        float x[N];
        Chunk<TYPE>::values(row.chunk(k), x);
        if (row.legal) {
            unsigned legal[N / 4];
            mask_words<N>(row.legal, row.head + k * N, row.actions, legal);
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = is_legal<N>(legal, i) ? x[i] : NONE;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) f(x[i]);
    }
    if (t < row.ends) f(row.at(row.end(t)));
}
template <int AT_ONCE, int TYPE> __device__ __forceinline__ float exact_max(const Row<TYPE>& row, int t, int threads) {
    float m = NONE;
    each_chunk<AT_ONCE>(row, t, threads, [&](float x) { m = fmaxf(m, x); });
    return warp_max(m);
}
template <int AT_ONCE, int TYPE> __device__ __forceinline__ Part exact_sums(const Row<TYPE>& row, float m, float scale, int t, int threads) {
    const float from = m == NONE ? 0.0f : m;
    Part p{m, 0.0f, 0.0f};
    each_chunk<AT_ONCE>(row, t, threads, [&](float x) {
        const float y = (x - from) * scale * LOG2E, e = exp2_fast(y);
        p.s += e;
        p.t += e > 0.0f ? y * e : 0.0f;
    });
#pragma unroll
    for (int by = 16; by; by /= 2) { p.s += __shfl_xor_sync(ALL, p.s, by); p.t += __shfl_xor_sync(ALL, p.t, by); }
    return p;
}
// The best of a row by one warp that goes through all its values, 32 at a time.
template <int TYPE> __device__ __forceinline__ unsigned long long best_of_all(const Row<TYPE>& row, int first, int step, unsigned lane, int top) {
    unsigned long long best = 0ull;
    for (int j0 = first; j0 < row.actions; j0 += step) {
        const int j = j0 + (int)lane;
        const float x = j < row.actions ? row.at(j) : NONE;
        take32(best, x > NONE ? order_key(x, (unsigned)j) : 0ull, lane, top);
    }
    return best;
}
// How many of n keys are larger than this one: its place in the order.
__device__ __forceinline__ int place_of(unsigned long long key, const unsigned long long* keys, int n) {
    int place = 0;
    for (int l = 0; l < n; ++l) place += keys[l] > key ? 1 : 0;
    return place;
}

// A chunk's values with the masked ones at minus infinity, their maximum, then all of them at FLOOR at least.  (bf16 without a mask goes there two values at a time,
// before the maximum: it is FLOOR then where there is nothing.)
template <int TYPE, bool MASKED>
__device__ __forceinline__ void take_chunk(const uint4& raw, const unsigned (&legal)[Chunk<TYPE>::N / 4], float (&x)[Chunk<TYPE>::N], float& m) {
    constexpr int N = Chunk<TYPE>::N;
    constexpr bool EARLY = TYPE == CUDARL_BF16 && !MASKED;
    if constexpr (EARLY) Chunk<TYPE>::floored(raw, x);
    else Chunk<TYPE>::values(raw, x);
    if constexpr (MASKED) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = is_legal<N>(legal, i) ? x[i] : NONE;
    }
#pragma unroll
    for (int i = 0; i < N; i += 2) m = max3(m, x[i], x[i + 1]);
    if constexpr (!EARLY) {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = max_nan(x[i], FLOOR);
    }
}
template <int TYPE> __device__ __forceinline__ void add_chunk(const float (&x)[Chunk<TYPE>::N], Two c2, Two mc2, Two& s2, Two& t2) {
#pragma unroll
    for (int i = 0; i < Chunk<TYPE>::N; i += 2) {
        const Two y2 = fma2(two(x[i], x[i + 1]), c2, mc2);
        float y0, y1;
        apart(y2, y0, y1);
        const Two e2 = two(exp2_fast(y0), exp2_fast(y1));
        s2 = add2(s2, e2);
        t2 = fma2(y2, e2, t2);
    }
}

// ------------------------------------------------------------------------------------------------------------------ rows of a warp
// A warp a row, the whole row in registers: CHUNKS pieces of 16 bytes a lane, and an end.  What is
// scalar in a row -- the taken action's logit, logarithm, quotient, addresses, the writes -- is done for up to 32 consecutive rows at a time, a lane each.
// The alternatives: the `top`-th largest of the lanes' maxima is a bound that `top` values reach; what reaches it is listed, and each of those counts how many
// are larger.  With about 28 of them and more the bound is so low that often more than WARP_KEYS values reach it, and the row is gone through by best_of_all, 32 values at
// a time: 100,000 x 1000 fp32 with 0 / 4 / 16 / 24 / 28 / 32 alternatives 75 / 117 / 187 / 286 / 717 / 1161 us.
// 65,536 x 257 fp32: 25 us (209 instructions a row), with a mask 40 (310), with a mask and 4 alternatives 65 (618, 0.63 issued per scheduler and cycle; a warp waits for
// its row's loads 3.4 and for fixed latencies 3.0 times as long as it issues).  257 values are 64 chunks and an end, and go through a kernel for twice as many: half of
// its places are empty.  (100,000 x 1000 fp32 with 4 alternatives 119 us, by the kernel for long rows 150; without 76 and 72.  Loading the next row into registers ahead, or having it
// fetched to L2, made it slower: 92 and 78 us.)
constexpr int WARP_KEYS = 64, GROUP_KEYS = 128;
// Blocks on an SM for which the registers suffice.
constexpr int warp_blocks(int values) { return values <= 8 ? 5 : values <= 16 ? 4 : 3; }

template <int TYPE, int CHUNKS, bool MASKED, bool TOP>
__global__ void __launch_bounds__(256, warp_blocks(CHUNKS * Chunk<TYPE>::N)) k_warp(Rows p, Outputs o, int group, bool alike) {
    using C = Chunk<TYPE>;
    constexpr int N = C::N;
    __shared__ unsigned long long keys_all[TOP ? 8 * WARP_KEYS : 1], sorted_all[TOP ? 8 * GROUP_KEYS : 1];
    const unsigned lane = threadIdx.x % 32u, warp = threadIdx.x / 32u;
    unsigned long long* const keys = keys_all + (TOP ? warp * WARP_KEYS : 0u);
    unsigned long long* const sorted = sorted_all + (TOP ? warp * GROUP_KEYS : 0u);                 // group * top <= GROUP_KEYS
    const float c = p.scale * LOG2E;
    const long long step = (long long)gridDim.x * 8 * group;
    long long first = ((long long)blockIdx.x * 8 + warp) * group;
    Row<TYPE> row(p, first < p.rows ? first : 0);
    for (; first < p.rows; first += step) {
        const int rows = (int)min((long long)group, p.rows - first);
        int a = -1;
        float xa = NONE;
        if ((int)lane < rows && p.taken) {
            a = __ldg(p.taken + first + lane);
            if ((unsigned)a < (unsigned)p.actions) {
                const long long r = first + lane;
                xa = p.legal && !__ldg(p.legal + r * p.legal_stride + a) ? NONE : Of<TYPE>::get(static_cast<const typename Of<TYPE>::T*>(p.logits)[r * p.stride + a]);
            }
        }
        Part mine{NONE, 0.0f, 0.0f};                                         // of the lane's row
        for (int i_row = 0; i_row < rows; ++i_row) {
            if (alike) row.move_to(p, first + i_row); else row = Row<TYPE>(p, first + i_row);
            uint4 raw[CHUNKS];
            unsigned legal[CHUNKS][N / 4];
#pragma unroll
            for (int u = 0; u < CHUNKS; ++u) {
                const int k = (int)lane + 32 * u;
                raw[u] = k < row.chunks ? row.chunk(k) : C::fill();
                if constexpr (MASKED) {
#pragma unroll
                    for (int i = 0; i < N / 4; ++i) legal[u][i] = 0u;
                    if (k < row.chunks) mask_words<N>(row.legal, row.head + k * N, row.actions, legal[u]);
                }
            }
            const float xe = (int)lane < row.ends ? row.at(row.end((int)lane)) : NONE;
            float x[CHUNKS][N], high[CHUNKS], m = fmaxf(xe, NONE);
#pragma unroll
            for (int u = 0; u < CHUNKS; ++u) {
                high[u] = NONE;
                take_chunk<TYPE, MASKED>(raw[u], legal[u], x[u], high[u]);
                m = fmaxf(m, high[u]);
            }
            const float own = m;
            m = warp_max(m);
            Part part{m, 0.0f, 0.0f};
            if (is_usual(m, c) || m == NONE) {
                const float mc = base_of(m, c), ye = fmaf(max_nan(xe, FLOOR), c, -mc), ee = exp2_fast(ye);
                const Two c2 = two(c, c), mc2 = two(-mc, -mc);
                Two s2 = two(ee, 0.0f), t2 = two(ye * ee, 0.0f);
#pragma unroll
                for (int u = 0; u < CHUNKS; ++u) add_chunk<TYPE>(x[u], c2, mc2, s2, t2);
                part.s = sum2(s2); part.t = sum2(t2);
#pragma unroll
                for (int by = 16; by; by /= 2) { part.s += __shfl_xor_sync(ALL, part.s, by); part.t += __shfl_xor_sync(ALL, part.t, by); }
            } else {                                                         // beyond the limit
                m = exact_max<1>(row, (int)lane, 32);
                part = exact_sums<1>(row, m, p.scale, (int)lane, 32);
            }
            if ((int)lane == i_row) mine = part;
            if constexpr (TOP) {
                const bool bad = !(part.s == part.s);
                const float bound = warp_ranked(own, o.top);
                int n = 0;
                if (bound > ABOVE_FLOOR && !bad) {
                    auto list = [&](float v, int j) {
                        const unsigned who = __ballot_sync(ALL, v >= bound);
                        if (!who) return;
                        const int place = n + __popc(who & ((1u << lane) - 1u));
                        if (v >= bound && place < WARP_KEYS) keys[place] = order_key(v, (unsigned)j);
                        n += __popc(who);
                    };
#pragma unroll
                    for (int u = 0; u < CHUNKS; ++u)
                        if (__any_sync(ALL, high[u] >= bound)) {
#pragma unroll
                            for (int i = 0; i < N; ++i) list(x[u][i], row.head + ((int)lane + 32 * u) * N + i);
                        }
                    list(xe, row.end((int)lane));
                    __syncwarp();
                }
                if (n >= o.top && n <= WARP_KEYS) {
                    for (int l = (int)lane; l < n; l += 32) {
                        const unsigned long long key = keys[l];
                        const int place = place_of(key, keys, n);
                        if (place < o.top) sorted[i_row * o.top + place] = key;
                    }
                } else {
                    const unsigned long long best = bad || part.s == 0.0f ? 0ull : best_of_all(row, 0, 32, lane, o.top);
                    if ((int)lane < o.top) sorted[i_row * o.top + (int)lane] = best;
                }
                __syncwarp();
            }
        }
        const Known known(mine);
        if ((int)lane < rows) {
            known.write(o, first + lane);
            if (o.logprob) o.logprob[first + lane] = known.bad ? known.log2_s : (unsigned)a < (unsigned)p.actions ? known.logprob(xa, p) : 0.0f;
        }
        if constexpr (TOP) {
            for (int l0 = 0; l0 < rows * o.top; l0 += 32) {
                const int l = l0 + (int)lane, of = min(l / o.top, 31);
                Known its = known;                                           // of the row that the place belongs to
                its.m = __shfl_sync(ALL, known.m, of); its.log2_s = __shfl_sync(ALL, known.log2_s, of);
                its.nothing = __shfl_sync(ALL, known.nothing, of); its.bad = __shfl_sync(ALL, known.bad, of);
                if (l < rows * o.top) write_top(o, p, its, first, l, sorted[l]);
            }
            __syncwarp();
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------ long rows
// T threads a row: a warp, 128, or the blocks of a cluster for few rows (which: launch_rows).  A thread takes batches of UNROLL chunks; a batch costs one maximum and one rebasing of the thread's
// sums.  The threads' parts are joined by shuffles, in shared memory, and over the cluster in the other blocks' shared memory.
//
// Alternatives: the maximum of every batch (of every GROUP of batches, for very long rows) is kept in shared memory.  32 of the threads' maxima, the largest of each
// warp, are values of the row, so the `top`-th largest of them is a bound that `top` values reach.  Only batches that reach it are read again -- a few dozen --
// and of what reaches the bound there each counts how many are larger.  Where too much does (rows of equal values) or too little (fewer than `top` values above
// FLOOR), every value of the row is gone through again, each warp with its 32 best in registers.
//
// With 128 threads the next batch is loaded ahead into registers (4096 x 131072 bf16: 179 us, without 195; a ring of bulk copies by one more warp: 186 to 210, and 262
// to 300 with alternatives, whose second look then waits for the copies' place).  Where the registers do not suffice for that it is fetched to L2 (with / without:
// 30000 x 4096 fp32 76 / 79 us, 20000 x 2500 f16, 4 alternatives 51 / 53).
constexpr int UNROLL = 4,  TABLE_ROWS = 32, LIST = 192, CANDIDATES = 256;

template <int T> struct Shared {
    Part part[T / 32];
    float high[32];                      // of the warps' threads, the 32 / (T / 32) largest of each
    float block_high[32];                // of those the 32 / blocks largest
    Part block;                          // of this block, for the other blocks of the cluster
    unsigned listed, found;
    unsigned list[LIST];
    unsigned long long key[CANDIDATES];
};
template <int T> __device__ __forceinline__ void team_sync() {
    if constexpr (T == 32) __syncwarp();
    else __syncthreads();
}
// The lane's place among the 32 lanes' values, of equal ones the lower lane first.
__device__ __forceinline__ int place_in_warp(float v, unsigned lane) {
    int place = 0;
#pragma unroll
    for (unsigned l = 0; l < 32u; ++l) {
        const float other = __shfl_sync(ALL, v, l);
        place += other > v || (other == v && l < lane) ? 1 : 0;
    }
    return place;
}

template <int TYPE, int T, bool MASKED, bool TOP>
__global__ void __launch_bounds__(T, (T == 128 && !MASKED ? 768 : 1024) / T) k_long(Rows p, Outputs o, int blocks, int group) {
    using C = Chunk<TYPE>;
    using Value = typename Of<TYPE>::T;
    constexpr int N = C::N, WARPS = T / 32, BATCH = UNROLL * T;
    constexpr bool AHEAD = T == 128 && !MASKED;                             // (with a mask the registers do not suffice)
    static_assert(WARPS * 32 <= CANDIDATES, "the warps' best have to fit");
    extern __shared__ __align__(128) unsigned char shared_bytes[];
    __shared__ Shared<T> sh;
    Value* const table = reinterpret_cast<Value*>(shared_bytes);
    const int t = (int)threadIdx.x, warp = t / 32;
    const unsigned lane = threadIdx.x % 32u;
    const int rank = blocks > 1 ? (int)(blockIdx.x % (unsigned)blocks) : 0;
    const float c = p.scale * LOG2E;
    const long long first = (long long)(blockIdx.x / (unsigned)blocks), step = gridDim.x / (unsigned)blocks;
    cg::cluster_group cluster = cg::this_cluster();
    for (long long r = first; r < p.rows; r += step) {
        const Row<TYPE> row(p, r);
        const int batches = (row.chunks + BATCH * blocks - 1) / (BATCH * blocks);      // of this block: the row's batch b * blocks + rank
        const int a = t == 0 && rank == 0 && p.taken ? __ldg(p.taken + r) : -1;
        const bool has_end = rank == 0 && t < row.ends;                      // (ends < 2 N <= 16 <= T)
        const float xe = has_end ? row.at(row.end(t)) : NONE;
        Part part{NONE, 0.0f, 0.0f};
        Two s2 = two(0.0f, 0.0f), t2 = s2;
        float high = NONE;                                                   // of the group of batches
        uint4 raw[UNROLL];
        unsigned legal[UNROLL][N / 4];
        auto load = [&](int b) {
            const int at = (b * blocks + rank) * BATCH + t;
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int k = at + u * T;
                raw[u] = k < row.chunks ? row.chunk(k) : C::fill();
                if constexpr (MASKED) {
#pragma unroll
                    for (int i = 0; i < N / 4; ++i) legal[u][i] = 0u;
                    if (k < row.chunks) mask_words<N>(row.legal, row.head + k * N, row.actions, legal[u]);
                }
            }
        };
        if (AHEAD) load(0);
        for (int b = 0; b < batches; ++b) {
            if (!AHEAD) load(b);
            if (!AHEAD && b + 1 < batches) {                                 // the next batch's bytes on their way to L2 meanwhile
                const int k = ((b + 1) * blocks + rank) * BATCH, left = min(BATCH, row.chunks - k) * N;
                const auto* const at = row.x + row.head + k * N;
                fetch_ahead(at, at + left, t, T);
                if (MASKED) fetch_ahead(row.legal + row.head + k * N, row.legal + row.head + k * N + left, t, T);
            }
            float x[UNROLL][N], bm = NONE;
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) take_chunk<TYPE, MASKED>(raw[u], legal[u], x[u], bm);
            if (AHEAD && b + 1 < batches) load(b + 1);
            if constexpr (TOP) {
                high = fmaxf(high, bm);
                if ((b + 1) % group == 0 || b + 1 == batches) { table[(b / group) * T + t] = Of<TYPE>::put(high); high = NONE; }
            }
            if (bm > part.m) {
                part.s += sum2(s2); part.t += sum2(t2);
                s2 = two(0.0f, 0.0f); t2 = s2;
                rebase(part, bm, c);
            }
            const Two c2 = two(c, c), mc2 = two(-base_of(part.m, c), -base_of(part.m, c));
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) add_chunk<TYPE>(x[u], c2, mc2, s2, t2);
        }
        part.s += sum2(s2); part.t += sum2(t2);
        if (has_end) take_one(part, xe, c);
        if constexpr (TOP) table[TABLE_ROWS * T + t] = Of<TYPE>::put(xe == xe ? xe : NONE);
        const float own = part.m;                                            // this thread's maximum

        join_lanes(part, c);
        if constexpr (TOP) {
            if constexpr (WARPS > 1) {
                constexpr int EACH = 32 / WARPS;
                float v = own;
                for (int k = 0; k < EACH; ++k) {
                    const float largest_left = warp_max(v);
                    if (lane == 0u) sh.high[warp * EACH + k] = largest_left;
                    if (lane == (unsigned)__ffs((int)__ballot_sync(ALL, v == largest_left)) - 1u) v = NONE;
                }
            }
            if (t == 0) sh.listed = sh.found = 0u;
        }
        if (lane == 0u) sh.part[warp] = part;
        team_sync<T>();
        float bound = FLOOR;
        if constexpr (TOP) bound = WARPS > 1 ? sh.high[lane] : own;          // 32 values of the row, one a lane
        if constexpr (T > 32) part = lane < WARPS ? sh.part[lane] : Part{NONE, 0.0f, 0.0f};
        if (T > 32 && blocks > 1) {
            if (warp == 0) {
                if constexpr (TOP) sh.block_high[place_in_warp(bound, lane)] = bound;
                join_lanes(part, c, WARPS);
                if (lane == 0u) sh.block = part;
            }
            cluster.sync();
            const Shared<T>* const other = cluster.map_shared_rank(&sh, (int)(lane % (unsigned)blocks));
            part = (int)lane < blocks ? other->block : Part{NONE, 0.0f, 0.0f};
            if constexpr (TOP) bound = other->block_high[lane / (unsigned)blocks];
        }
        if constexpr (TOP) bound = warp_min(place_in_warp(bound, lane) < o.top ? bound : INFINITY);
        float m = warp_max(part.m);
        if (is_usual(m, c) || m == NONE) {
            if constexpr (T > 32) join_lanes(part, c, blocks > 1 ? 8 : WARPS);
        } else {                                                             // beyond the limit; every block of a cluster goes through the whole row
            m = exact_max<4>(row, t, T);
            if constexpr (T > 32) {
                team_sync<T>();
                if (lane == 0u) sh.part[warp].m = m;
                team_sync<T>();
                m = warp_max(sh.part[lane % WARPS].m);
            }
            part = exact_sums<4>(row, m, p.scale, t, T);
            if constexpr (T > 32) {
                team_sync<T>();
                if (lane == 0u) sh.part[warp] = part;
                team_sync<T>();
                part = lane < WARPS ? sh.part[lane] : Part{m, 0.0f, 0.0f};
                for (int by = WARPS / 2; by; by /= 2) { part.s += __shfl_xor_sync(ALL, part.s, by); part.t += __shfl_xor_sync(ALL, part.t, by); }
            }
        }
        part.s = __shfl_sync(ALL, part.s, 0); part.t = __shfl_sync(ALL, part.t, 0); part.m = m;
        const Known known(part);
        if (t == 0 && rank == 0) {
            known.write(o, r);
            if (o.logprob) o.logprob[r] = known.bad ? known.log2_s : (unsigned)a >= (unsigned)row.actions ? 0.0f : known.logprob(row.at(a), p);
        }
        if constexpr (TOP) {
            // batches that reach the bound, then what reaches it in them: into the first block's list
            Shared<T>* const to = T > 32 && blocks > 1 ? cluster.map_shared_rank(&sh, 0) : &sh;
            const int rows_used = (batches + group - 1) / group;
            if (bound > ABOVE_FLOOR && own >= bound) {
                auto list_it = [&](int q) {
                    const unsigned place = atomicAdd(&sh.listed, 1u);
                    if (place < LIST) sh.list[place] = (unsigned)(q * T + t);
                    else atomicAdd(&to->found, CANDIDATES + 1u);             // too many
                };
                for (int q = 0; q < rows_used; ++q)
                    if (Of<TYPE>::get(table[q * T + t]) >= bound) list_it(q);
                if (xe >= bound) list_it(TABLE_ROWS);
            }
            team_sync<T>();
            // a thread a chunk of a listed batch, so that all of them are read again at the same time
            const int items = (int)min(sh.listed, (unsigned)LIST) * group * UNROLL;
            for (int l = t; l < items; l += T) {
                const int entry = (int)sh.list[l / (group * UNROLL)], q = entry / T, owner = entry % T, piece = l % (group * UNROLL);
                auto take = [&](float x, int j) {
                    if (x >= bound) {
                        const unsigned place = atomicAdd(&to->found, 1u);
                        if (place < CANDIDATES) to->key[place] = order_key(x, (unsigned)j);
                    }
                };
                if (q == TABLE_ROWS) {
                    if (piece == 0) take(row.at(row.end(owner)), row.end(owner));
                    continue;
                }
                const int b = q * group + piece / UNROLL, k = (b * blocks + rank) * BATCH + piece % UNROLL * T + owner;
                if (b >= batches || k >= row.chunks) continue;
                float x[N];
                C::floored(row.chunk(k), x);
                if constexpr (MASKED) {
                    unsigned legal[N / 4];
                    mask_words<N>(row.legal, row.head + k * N, row.actions, legal);
#pragma unroll
                    for (int i = 0; i < N; ++i) x[i] = is_legal<N>(legal, i) ? x[i] : FLOOR;
                }
#pragma unroll
                for (int i = 0; i < N; ++i) take(x[i], row.head + k * N + i);
            }
            if (T > 32 && blocks > 1) cluster.sync(); else team_sync<T>();
            if (rank == 0) {
                const unsigned n = sh.found;
                if (n >= (unsigned)o.top && n <= (unsigned)CANDIDATES && !known.bad) {
                    for (unsigned l = (unsigned)t; l < n; l += T) {
                        const unsigned long long key = sh.key[l];
                        const int place = place_of(key, sh.key, (int)n);
                        if (place < o.top) write_top(o, p, known, r, place, key);
                    }
                } else {
                    unsigned long long best = known.bad || known.nothing ? 0ull : best_of_all(row, warp * 32, T, lane, o.top);
                    if constexpr (T > 32) {
                        team_sync<T>();                                      // the list has been counted by all
                        sh.key[t] = best;
                        team_sync<T>();
                    }
                    if (warp == 0) {
                        for (int w = 1; w < WARPS; ++w) best = merged32(best, sh.key[w * 32 + lane], lane);
                        if ((int)lane < o.top) write_top(o, p, known, r, (int)lane, best);
                    }
                }
            }
        }
        if (T > 32 && blocks > 1) cluster.sync();                   // nobody leaves, or begins the next row, while its shared memory is read
        else team_sync<T>();
    }
}

// ------------------------------------------------------------------------------------------------------------------ gradient
// What one row's gradient needs besides its values:  dx = -p (A + B log2 p), and at the action taken scale (gl (1 - p) - gH p (ln p + H)) with 1 - p = -expm1(ln p).
struct Slope {
    float m, mc, log2_s, c, scale, A, B, gl, gh, h;
    int taken;
    bool exact, nothing, bad;
    __device__ __forceinline__ Slope(const Rows& p, const float4* stats, const float* grad_logprob, const float* grad_entropy, long long r) {
        const float4 st = __ldg(stats + r);
        const int a = p.taken ? __ldg(p.taken + r) : -1;
        taken = (unsigned)a < (unsigned)p.actions ? a : -1;
        gl = taken >= 0 && grad_logprob ? __ldg(grad_logprob + r) : 0.0f;
        gh = grad_entropy ? __ldg(grad_entropy + r) : 0.0f;
        scale = p.scale; c = scale * LOG2E;
        m = st.x; mc = m * c; log2_s = st.y; h = st.z;
        A = scale * (gl + gh * h); B = scale * gh * LN2;
        nothing = log2_s == NONE; bad = !(log2_s == log2_s);
        exact = !is_usual(m, c);
    }
    __device__ __forceinline__ bool usual() const { return !exact && !nothing && !bad; }
    // One value, whatever the row is like.
    __device__ __forceinline__ float one(float x, int j) const {
        if (nothing) return 0.0f;
        if (bad) return log2_s;
        const float lp = fmaxf((exact ? (x - m) * scale * LOG2E : fmaf(fmaxf(x, FLOOR), c, -mc)) - log2_s, FLOOR), pr = exp2_fast(lp);
        if (j == taken) return scale * (-gl * expm1f(lp * LN2) - gh * pr * fmaf(lp, LN2, h));
        return -pr * fmaf(B, lp, A);
    }
};

// Short rows have their sums in a few instructions: they are taken again instead of the statistics, which are as long as such a row.  AT_ONCE rows of a thread have
// their loads on their way together where a row is a single load.
template <int TYPE, int G, int E, bool WIDE>
__global__ void __launch_bounds__(256) k_short_backward(Rows p, const float* grad_logprob, const float* grad_entropy, void* grad, long long grad_stride) {
    using O = Of<TYPE>;
    constexpr int AT_ONCE = G == 1 && E == 4 ? 2 : 1, ROWS = 256 / G;
    const int lane = (int)threadIdx.x % G;
    const long long step = (long long)gridDim.x * ROWS * AT_ONCE;
    for (long long first = (long long)blockIdx.x * ROWS * AT_ONCE; first < p.rows; first += step) {
        float xs[AT_ONCE][E], gls[AT_ONCE], ghs[AT_ONCE];
        int as[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const long long mine = first + u * ROWS + (int)threadIdx.x / G, r = mine < p.rows ? mine : p.rows - 1;
            load_short<TYPE, G, E, WIDE>(p, r, lane, xs[u]);
            as[u] = p.taken ? __ldg(p.taken + r) : -1;
            gls[u] = grad_logprob ? __ldg(grad_logprob + r) : 0.0f;
            ghs[u] = grad_entropy ? __ldg(grad_entropy + r) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const long long mine = first + u * ROWS + (int)threadIdx.x / G, r = mine < p.rows ? mine : p.rows - 1;
            float (&x)[E] = xs[u];
            float y[E], e[E];
            const int a = as[u];
            const bool taken = (unsigned)a < (unsigned)p.actions;
            const float gl = taken ? gls[u] : 0.0f, gh = ghs[u];
            bool exact;
            const Part part = sum_short<G, E>(x, p.scale, y, e, exact);
            const Known known(part);
            const float A = -p.scale * (gl + gh * known.h), B = -p.scale * gh * LN2, share = __fdividef(1.0f, part.s);
            const float more = p.scale * gl;                                 // of the action taken: scale gl (1 - p) is one product less p's
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                const Two lp2 = add2(two(y[i], y[i + 1]), two(-known.log2_s, -known.log2_s)), p2 = mul2(two(e[i], e[i + 1]), two(share, share));
                apart(mul2(p2, fma2(two(B, B), lp2, two(A, A))), x[i], x[i + 1]);
            }
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] += taken && short_action<G, E, WIDE>(lane, i) == a ? more : 0.0f;
            if (known.nothing || known.bad) {
#pragma unroll
                for (int i = 0; i < E; ++i) x[i] = known.bad ? known.log2_s : 0.0f;
            }
            if (p.legal) {
                const unsigned char* legal = p.legal + r * p.legal_stride;
#pragma unroll
                for (int i = 0; i < E; ++i) { const int j = short_action<G, E, WIDE>(lane, i); if (j < p.actions && !__ldg(legal + j)) x[i] = 0.0f; }
            }
            if (mine >= p.rows) continue;                                    // (a whole team: nothing of it is waited for)
            auto* at = static_cast<typename O::T*>(grad) + r * grad_stride;
            constexpr int BYTES = E * (int)sizeof(typename O::T);
            if (WIDE && lane * E + E <= p.actions) {
                if constexpr (BYTES == 8 && TYPE != CUDARL_F32) *reinterpret_cast<uint2*>(at + lane * E) = make_uint2(Chunk<TYPE>::two16(x[0], x[1]), Chunk<TYPE>::two16(x[2], x[3]));
                else if constexpr (BYTES >= 16) {
#pragma unroll
                    for (int k = 0; k < BYTES / 16; ++k) {
                        float values[Chunk<TYPE>::N];
#pragma unroll
                        for (int i = 0; i < Chunk<TYPE>::N; ++i) values[i] = x[k * Chunk<TYPE>::N + i];
                        reinterpret_cast<uint4*>(at + lane * E)[k] = Chunk<TYPE>::pack(values);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i) { const int j = short_action<G, E, WIDE>(lane, i); if (j < p.actions) at[j] = O::put(x[i]); }
            }
        }
    }
}

// A chunk's gradient.
template <int TYPE>
__device__ __forceinline__ void slope_chunk(const Slope& slope, bool usual, const uint4& raw, int j0, float (&v)[Chunk<TYPE>::N]) {
    constexpr int N = Chunk<TYPE>::N;
    if (usual) {
        const Two c2 = two(slope.c, slope.c), mc2 = two(-slope.mc, -slope.mc), l2 = two(-slope.log2_s, -slope.log2_s), A2 = two(-slope.A, -slope.A), B2 = two(-slope.B, -slope.B);
        Chunk<TYPE>::floored(raw, v);
        const bool has = (unsigned)(slope.taken - j0) < (unsigned)N;
        float own = v[0];
        if (has) {
#pragma unroll
            for (int i = 1; i < N; ++i) own = slope.taken - j0 == i ? v[i] : own;
            own = slope.one(own, slope.taken);
        }
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const Two lp2 = add2(fma2(two(v[i], v[i + 1]), c2, mc2), l2);
            float a, b;
            apart(lp2, a, b);
            apart(mul2(two(exp2_fast(a), exp2_fast(b)), fma2(B2, lp2, A2)), v[i], v[i + 1]);
        }
        if (has) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = slope.taken - j0 == i ? own : v[i];
        }
    } else {
        Chunk<TYPE>::values(raw, v);
#pragma unroll 1
        for (int i = 0; i < N; ++i) {
            float one = v[0];
#pragma unroll
            for (int k = 1; k < N; ++k) one = i == k ? v[k] : one;
            one = slope.one(one, j0 + i);
#pragma unroll
            for (int k = 0; k < N; ++k) v[k] = i == k ? one : v[k];
        }
    }
}

// A warp a row, all its chunks at once.
template <int TYPE, int CHUNKS, bool MASKED>
__global__ void __launch_bounds__(256, warp_blocks(CHUNKS * Chunk<TYPE>::N)) k_warp_backward(Rows p, const float4* stats, const float* grad_logprob, const float* grad_entropy, void* grad,
                                                                                              long long grad_stride) {
    using C = Chunk<TYPE>;
    using O = Of<TYPE>;
    constexpr int N = C::N;
    const int lane = (int)threadIdx.x % 32;
    const long long step = (long long)gridDim.x * 8;
    for (long long r = (long long)blockIdx.x * 8 + (int)threadIdx.x / 32; r < p.rows; r += step) {
        const auto* x = static_cast<const typename O::T*>(p.logits) + r * p.stride;
        auto* g = static_cast<typename O::T*>(grad) + r * grad_stride;
        const unsigned char* legal = MASKED ? p.legal + r * p.legal_stride : nullptr;
        const int head = min((int)((16u - ((unsigned)reinterpret_cast<uintptr_t>(g) & 15u)) & 15u) / (int)sizeof(typename O::T), p.actions);
        const int chunks = (p.actions - head) / N, ends = p.actions - chunks * N;
        const bool together = (((unsigned)reinterpret_cast<uintptr_t>(x) ^ (unsigned)reinterpret_cast<uintptr_t>(g)) & 15u) == 0u;
        uint4 raw[CHUNKS];
        unsigned mask[CHUNKS][N / 4];
#pragma unroll
        for (int u = 0; u < CHUNKS; ++u) {
            const int k = lane + 32 * u;
            raw[u] = C::fill();
            if (k < chunks) {
                raw[u] = together ? *reinterpret_cast<const uint4*>(x + head + k * N) : gather_chunk(x + head + k * N);
                if constexpr (MASKED) mask_words<N>(legal, head + k * N, p.actions, mask[u]);
            }
        }
        const Slope slope(p, stats, grad_logprob, grad_entropy, r);
        const bool usual = slope.usual();
        if (lane < ends) {
            const int j = lane < head ? lane : chunks * N + lane;
            g[j] = O::put(MASKED && !__ldg(legal + j) ? 0.0f : slope.one(O::get(x[j]), j));
        }
#pragma unroll
        for (int u = 0; u < CHUNKS; ++u) {
            const int k = lane + 32 * u;
            if (k >= chunks) continue;
            float v[N];
            slope_chunk<TYPE>(slope, usual, raw[u], head + k * N, v);
            if constexpr (MASKED) {
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = is_legal<N>(mask[u], i) ? v[i] : 0.0f;
            }
            *reinterpret_cast<uint4*>(g + head + k * N) = C::pack(v);
        }
    }
}

// Long rows: a block takes UNROLL chunks a thread of a piece of a row; chunks begin where the gradient's address is aligned, and the logits are read in the same
// chunks where their address is too, else one by one.
constexpr int PIECE_THREADS = 128;
template <int TYPE, bool MASKED>
__global__ void __launch_bounds__(PIECE_THREADS) k_long_backward(Rows p, const float4* stats, const float* grad_logprob, const float* grad_entropy, void* grad, long long grad_stride) {
    using C = Chunk<TYPE>;
    using O = Of<TYPE>;
    constexpr int N = C::N;
    const int t = (int)threadIdx.x, T = (int)blockDim.x;
    for (long long r = blockIdx.y; r < p.rows; r += gridDim.y) {
        const auto* x = static_cast<const typename O::T*>(p.logits) + r * p.stride;
        auto* g = static_cast<typename O::T*>(grad) + r * grad_stride;
        const unsigned char* legal = MASKED ? p.legal + r * p.legal_stride : nullptr;
        const int head = min((int)((16u - ((unsigned)reinterpret_cast<uintptr_t>(g) & 15u)) & 15u) / (int)sizeof(typename O::T), p.actions);
        const int chunks = (p.actions - head) / N, ends = p.actions - chunks * N;
        const bool together = (((unsigned)reinterpret_cast<uintptr_t>(x) ^ (unsigned)reinterpret_cast<uintptr_t>(g)) & 15u) == 0u;
        const int base = (int)blockIdx.x * UNROLL * T + t;
        uint4 raw[UNROLL];
        unsigned mask[UNROLL][N / 4];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int k = base + u * T;
            raw[u] = C::fill();
            if (k < chunks) {
                raw[u] = together ? *reinterpret_cast<const uint4*>(x + head + k * N) : gather_chunk(x + head + k * N);
                if constexpr (MASKED) mask_words<N>(legal, head + k * N, p.actions, mask[u]);
            }
        }
        const Slope slope(p, stats, grad_logprob, grad_entropy, r);
        const bool usual = slope.usual();
        if (blockIdx.x == 0u && t < ends) {
            const int j = t < head ? t : chunks * N + t;
            g[j] = O::put(MASKED && !__ldg(legal + j) ? 0.0f : slope.one(O::get(x[j]), j));
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int k = base + u * T;
            if (k >= chunks) continue;
            float v[N];
            slope_chunk<TYPE>(slope, usual, raw[u], head + k * N, v);
            if constexpr (MASKED) {
#pragma unroll
                for (int i = 0; i < N; ++i) v[i] = is_legal<N>(mask[u], i) ? v[i] : 0.0f;
            }
            *reinterpret_cast<uint4*>(g + head + k * N) = C::pack(v);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------ calls
int check_rows(const cudarl_policy_rows* p) {
    if (!p) return fail_global(-1, "null argument");
    if (p->struct_size != sizeof(cudarl_policy_rows)) return fail_global(-1, "cudarl_policy_rows.struct_size mismatch");
    if (p->type != CUDARL_F32 && p->type != CUDARL_BF16 && p->type != CUDARL_F16) return fail_global(-1, "type must be CUDARL_F32, CUDARL_BF16 or CUDARL_F16");
    if (p->rows < 0 || p->actions < 1 || p->actions > CUDARL_MAX_POLICY_ACTIONS) return fail_global(-1, "rows or actions out of range");
    if (p->row_stride < p->actions) return fail_global(-1, "row_stride smaller than a row");
    if (p->legal && p->legal_stride != 0 && p->legal_stride < p->actions) return fail_global(-1, "legal_stride must be 0 or at least a row");
    const int64_t widest = p->row_stride > p->legal_stride ? p->row_stride : p->legal_stride;
    if (p->rows > (1ll << 40) || widest > (1ll << 40) || p->rows > (1ll << 56) / widest) return fail_global(-1, "rows or strides out of range");
    if (!(p->inv_temperature >= 1e-6f && p->inv_temperature <= 1e6f)) return fail_global(-1, "inv_temperature must be in 1e-6 .. 1e6");
    if (p->rows > 0 && !p->logits) return fail_global(-1, "null logits");
    return 0;
}

Rows device_rows(const cudarl_policy_rows* p) {
    return Rows{p->logits, p->legal, p->taken, (long long)p->rows, (long long)p->row_stride, (long long)p->legal_stride, (int)p->actions, p->inv_temperature};
}

unsigned blocks_of(long long work, int each) {                               // more work than that is done in turns
    const long long n = (work + each - 1) / each;
    return (unsigned)(n < (1ll << 28) ? n : (1ll << 28));
}
bool aligned_rows(const void* base, long long stride, int value, int bytes) {
    return reinterpret_cast<uintptr_t>(base) % (unsigned)bytes == 0 && stride * value % bytes == 0;
}

constexpr int SHORT_ACTIONS = CUDARL_ACTIONS_WITHOUT_STATS, WARP_ACTIONS = 1024;

template <int TYPE, int G, int E, bool WIDE>
cudaError_t launch_short(const Rows& p, const Outputs& o, cudaStream_t st) {
    const unsigned grid = blocks_of(p.rows, 256 / G);
    return o.top ? launch(k_short<TYPE, G, E, WIDE, true>, grid, 256, st, p, o) : launch(k_short<TYPE, G, E, WIDE, false>, grid, 256, st, p, o);
}
struct BackwardArgs { const float4* stats; const float* gl; const float* gh; void* grad; long long stride; };
template <int TYPE, int G, int E, bool WIDE>
cudaError_t launch_short(const Rows& p, const BackwardArgs& b, cudaStream_t st) {
    return launch(k_short_backward<TYPE, G, E, WIDE>, blocks_of(p.rows, 256 / G * (G == 1 && E == 4 ? 2 : 1)), 256, st, p, b.gl, b.gh, b.grad, b.stride);
}
// Rows of up to SHORT_ACTIONS actions, either way (a call's outputs or a gradient's arguments).
template <int TYPE, class Args>
cudaError_t launch_short(const Rows& p, const Args& args, bool wide4, bool wide8, cudaStream_t st) {
    const int v = p.actions;
    if (v <= 4 && wide4) return launch_short<TYPE, 1, 4, true>(p, args, st);
    if (v <= 8) return wide8 ? launch_short<TYPE, 1, 8, true>(p, args, st) : launch_short<TYPE, 4, 2, false>(p, args, st);
    if (v <= 16) return wide8 ? launch_short<TYPE, 2, 8, true>(p, args, st) : launch_short<TYPE, 4, 4, false>(p, args, st);
    if (v <= 32) return wide8 ? launch_short<TYPE, 4, 8, true>(p, args, st) : launch_short<TYPE, 4, 8, false>(p, args, st);
    if (v <= 64) return wide8 ? launch_short<TYPE, 8, 8, true>(p, args, st) : launch_short<TYPE, 8, 8, false>(p, args, st);
    return wide8 ? launch_short<TYPE, 16, 8, true>(p, args, st) : launch_short<TYPE, 16, 8, false>(p, args, st);
}

template <int TYPE, int VALUES>
cudaError_t launch_warp(const Rows& p, const Outputs& o, int sms, cudaStream_t st) {
    constexpr int CHUNKS = VALUES / 32 / Chunk<TYPE>::N;
    const unsigned most = (unsigned)(sms * warp_blocks(VALUES / 32));
    // as many rows for a warp at a time as leave every warp of the GPU some
    int group = 1;
    while (group < 32 && group * 2 * (o.top ? o.top : 1) <= GROUP_KEYS && p.rows >= 16ll * group * most) group *= 2;
    const bool alike = p.stride * (long long)sizeof(typename Of<TYPE>::T) % 16 == 0;
    const unsigned all = blocks_of(p.rows, 8 * group), grid = all < most ? all : most;
    if (p.legal) return o.top ? launch(k_warp<TYPE, CHUNKS, true, true>, grid, 256, st, p, o, group, alike) : launch(k_warp<TYPE, CHUNKS, true, false>, grid, 256, st, p, o, group, alike);
    return o.top ? launch(k_warp<TYPE, CHUNKS, false, true>, grid, 256, st, p, o, group, alike) : launch(k_warp<TYPE, CHUNKS, false, false>, grid, 256, st, p, o, group, alike);
}
template <int TYPE, int VALUES>
cudaError_t launch_warp(const Rows& p, const BackwardArgs& b, int sms, cudaStream_t st) {
    constexpr int CHUNKS = VALUES / 32 / Chunk<TYPE>::N;
    const unsigned most = (unsigned)(sms * warp_blocks(VALUES / 32)), all = blocks_of(p.rows, 8), grid = all < most ? all : most;
    return launch(p.legal ? k_warp_backward<TYPE, CHUNKS, true> : k_warp_backward<TYPE, CHUNKS, false>, grid, 256, st, p, b.stats, b.gl, b.gh, b.grad, b.stride);
}

template <int TYPE, int T, bool MASKED, bool TOP>
cudaError_t launch_long(const Rows& p, const Outputs& o, int blocks, cudaStream_t st) {
    const long long batch = (long long)UNROLL * T * blocks, chunks = p.actions / Chunk<TYPE>::N;
    const int group = (int)((chunks + batch * TABLE_ROWS) / (batch * TABLE_ROWS));
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(T);
    cfg.dynamicSmemBytes = TOP ? (size_t)(TABLE_ROWS + 1) * T * sizeof(typename Of<TYPE>::T) : 0;
    cfg.stream = st;
    cfg.gridDim = dim3((unsigned)((p.rows < (1ll << 26) ? p.rows : (1ll << 26)) * blocks));
    cudaLaunchAttribute attr[1];
    if (blocks > 1) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)blocks; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr; cfg.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&cfg, k_long<TYPE, T, MASKED, TOP>, p, o, blocks, group);
}
template <int TYPE, int T>
cudaError_t launch_long(const Rows& p, const Outputs& o, int blocks, cudaStream_t st) {
    if (p.legal) return o.top ? launch_long<TYPE, T, true, true>(p, o, blocks, st) : launch_long<TYPE, T, true, false>(p, o, blocks, st);
    return o.top ? launch_long<TYPE, T, false, true>(p, o, blocks, st) : launch_long<TYPE, T, false, false>(p, o, blocks, st);
}

template <int TYPE>
cudaError_t launch_rows(const Rows& p, const Outputs& o, int sms, cudaStream_t st) {
    constexpr int value = (int)sizeof(typename Of<TYPE>::T);
    const int v = p.actions;
    if (v <= SHORT_ACTIONS) return launch_short<TYPE>(p, o, aligned_rows(p.logits, p.stride, value, 4 * value), aligned_rows(p.logits, p.stride, value, 16), st);
    if (v <= 256) return launch_warp<TYPE, 256>(p, o, sms, st);
    if (v <= 512) return launch_warp<TYPE, 512>(p, o, sms, st);
    if (v <= WARP_ACTIONS) return launch_warp<TYPE, 1024>(p, o, sms, st);
    // a cluster for each row where there are too few rows to occupy the GPU, as long as each block still gets a batch (bf16, 20 alternatives, 1 / 2 / 4 / 8 blocks a
    // row: 1 x 131072 32 / 20 / 16 / 14 us, 74 rows 34 / 21 / 19 / 25, 200 rows 34 / 26 / 32 / 40)
    int blocks = 1;
    while (blocks < 8 && p.rows * blocks < 2ll * sms && (long long)v >= 256ll * Chunk<TYPE>::N * UNROLL * blocks) blocks *= 2;
    if (blocks > 1) return launch_long<TYPE, 256>(p, o, blocks, st);
    // a warp for each row where there are enough of them to occupy the GPU and what is done once a row weighs more than the wait for a batch (a warp / 128 threads:
    // 8192 x 8192 bf16, 4 alternatives 44 / 61 us, 20000 x 2500 f16 53 / 113; 600 x 30000 fp32 50 / 24, 2047 x 65537 bf16 71 / 57)
    if (v <= 8192 && p.rows >= 8ll * sms) return launch_long<TYPE, 32>(p, o, 1, st);
    return launch_long<TYPE, 128>(p, o, 1, st);
}

template <int TYPE>
cudaError_t launch_backward(const Rows& p, const BackwardArgs& b, int sms, cudaStream_t st) {
    constexpr int value = (int)sizeof(typename Of<TYPE>::T);
    const int v = p.actions;
    if (v <= SHORT_ACTIONS)
        return launch_short<TYPE>(p, b, aligned_rows(p.logits, p.stride, value, 4 * value) && aligned_rows(b.grad, b.stride, value, 4 * value),
                                  aligned_rows(p.logits, p.stride, value, 16) && aligned_rows(b.grad, b.stride, value, 16), st);
    if (v <= 256) return launch_warp<TYPE, 256>(p, b, sms, st);
    if (v <= 512) return launch_warp<TYPE, 512>(p, b, sms, st);
    if (v <= WARP_ACTIONS) return launch_warp<TYPE, 1024>(p, b, sms, st);
    // as few pieces a row as PIECE_THREADS a block allow, and no more threads in a block than a piece has work for (always 256 threads / as here: 20000 x 2500 f16
    // 67 / 43 us, 40000 x 1500 bf16 113 / 50; at most 256 / 128: 20000 x 6000 bf16 86 / 82, 10000 x 9000 masked 105 / 86, 20000 x 2500 fp32 63.5 / 67.6)
    const int chunks = v / Chunk<TYPE>::N, most = PIECE_THREADS * UNROLL, pieces = (chunks + most - 1) / most, each = (chunks + pieces * UNROLL - 1) / (pieces * UNROLL);
    const int threads = each <= 64 ? 64 : (each + 31) / 32 * 32;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)pieces, (unsigned)(p.rows < 65535 ? p.rows : 65535)); cfg.blockDim = dim3((unsigned)threads); cfg.stream = st;
    return cudaLaunchKernelEx(&cfg, p.legal ? k_long_backward<TYPE, true> : k_long_backward<TYPE, false>, p, b.stats, b.gl, b.gh, b.grad, b.stride);
}

}  // namespace

extern "C" int cudarl_policy_logprobs(const cudarl_policy_rows* p, float* logprob, float* entropy, float* stats, int32_t top, int32_t* top_actions,
                                      float* top_logprobs, void* stream) {
    int rc = check_rows(p);
    if (rc) return rc;
    if (top < 0 || top > CUDARL_MAX_TOP) return fail_global(-1, "top out of range (0 .. CUDARL_MAX_TOP)");
    if (top > 0 && p->rows > 0 && (!top_actions || !top_logprobs)) return fail_global(-1, "top without both of its arrays");
    if (logprob && p->rows > 0 && !p->taken) return fail_global(-1, "logprob without the actions taken");
    if (p->rows == 0) return 0;
    if (!logprob && !entropy && !stats && !top) return fail_global(-1, "no output");
    CallerArrays arrays;
    if ((rc = arrays.check("logits", p->logits, type_bytes(p->type))) || (rc = arrays.check_if("legal", p->legal, 1)) || (rc = arrays.check_if("taken", p->taken, 4)) ||
        (rc = arrays.check_if("logprob", logprob, 4)) || (rc = arrays.check_if("entropy", entropy, 4)) || (rc = arrays.check_if("stats", stats, 16))) return rc;
    if (top && ((rc = arrays.check("top_actions", top_actions, 4)) || (rc = arrays.check("top_logprobs", top_logprobs, 4)))) return rc;
    CurrentDevice current;
    int sms = 0;
    cudaError_t e = current.set(arrays.device());
    if (e == cudaSuccess) e = multiprocessors(&sms);
    if (e != cudaSuccess) return fail_cuda("cudarl_policy_logprobs", e);
    const Rows r = device_rows(p);
    const Outputs o{logprob, entropy, reinterpret_cast<float4*>(stats), top_actions, top_logprobs, top};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    e = p->type == CUDARL_F32 ? launch_rows<CUDARL_F32>(r, o, sms, st) : p->type == CUDARL_BF16 ? launch_rows<CUDARL_BF16>(r, o, sms, st) : launch_rows<CUDARL_F16>(r, o, sms, st);
    return e == cudaSuccess ? 0 : fail_cuda("cudarl_policy_logprobs", e);
}

extern "C" int cudarl_policy_logprobs_backward(const cudarl_policy_rows* p, const float* stats, const float* grad_logprob, const float* grad_entropy,
                                               void* grad_logits, int64_t grad_stride, void* stream) {
    int rc = check_rows(p);
    if (rc) return rc;
    if (grad_stride < p->actions || grad_stride > (1ll << 40) || p->rows > (1ll << 56) / grad_stride) return fail_global(-1, "grad_stride smaller than a row, or out of range");
    if (p->rows == 0) return 0;
    if (!stats || !grad_logits) return fail_global(-1, "null stats or grad_logits");
    if (grad_logprob && !p->taken) return fail_global(-1, "grad_logprob without the actions taken");
    if (grad_logits == p->logits && grad_stride != p->row_stride) return fail_global(-1, "gradients in the logits' place need the logits' stride");
    CallerArrays arrays;
    const size_t align = type_bytes(p->type);
    if ((rc = arrays.check("logits", p->logits, align)) || (rc = arrays.check_if("legal", p->legal, 1)) || (rc = arrays.check_if("taken", p->taken, 4)) ||
        (p->actions > SHORT_ACTIONS && (rc = arrays.check("stats", stats, 16))) || (rc = arrays.check_if("grad_logprob", grad_logprob, 4)) || (rc = arrays.check_if("grad_entropy", grad_entropy, 4)) ||
        (rc = arrays.check("grad_logits", grad_logits, align))) return rc;
    CurrentDevice current;
    int sms = 0;
    cudaError_t e = current.set(arrays.device());
    if (e == cudaSuccess) e = multiprocessors(&sms);
    if (e != cudaSuccess) return fail_cuda("cudarl_policy_logprobs_backward", e);
    const Rows r = device_rows(p);
    const BackwardArgs b{reinterpret_cast<const float4*>(stats), grad_logprob, grad_entropy, grad_logits, (long long)grad_stride};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    e = p->type == CUDARL_F32 ? launch_backward<CUDARL_F32>(r, b, sms, st) : p->type == CUDARL_BF16 ? launch_backward<CUDARL_BF16>(r, b, sms, st) : launch_backward<CUDARL_F16>(r, b, sms, st);
    return e == cudaSuccess ? 0 : fail_cuda("cudarl_policy_logprobs_backward", e);
}
