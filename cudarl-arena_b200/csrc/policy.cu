// policy.cu -- log probabilities of the actions taken, entropy and most probable alternatives of rows of logits, and the gradient of the logits.
//
// Row x, legal actions L, scale = 1 / temperature, m = max x.  In base 2, with c = scale log2(e):
//   y = x c - m c <= 0,   S = sum 2^y,   log2 p = y - log2 S,   H = ln 2 (log2 S - (sum y 2^y) / S)      (both terms >= 0: nothing cancels)
//   dx_j = scale (gl ([j = taken] - p_j) - gH p_j (ln p_j + H))
// What a row leaves for its gradient: {m, log2 S, H}.
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
// Larger for the larger logit, of equal ones for the lower action; 0 for none.
__device__ __forceinline__ unsigned long long order_key(float x, unsigned action) {
    const unsigned b = __float_as_uint(x + 0.0f);                            // -0 counts as 0
    return ((unsigned long long)((b & 0x80000000u) ? ~b : b | 0x80000000u) << 32) | (0xFFFFFFFFu - action);
}
__device__ __forceinline__ float key_value(unsigned long long key) {
    const unsigned b = (unsigned)(key >> 32);
    return __uint_as_float((b & 0x80000000u) ? b & 0x7FFFFFFFu : ~b);
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
    const float y = fmaf(x, c, -base_of(p.m, c)), e = exp2_fast(y);
    p.s += e;
    p.t = fmaf(y, e, p.t);
}
__device__ __forceinline__ void join(Part& a, Part b, float c) {
    const float m = fmaxf(a.m, b.m);
    rebase(a, m, c); rebase(b, m, c);
    a.s += b.s; a.t += b.t;
}

// What is known of a whole row.
struct Known {
    float m, log2_s, h;
    bool nothing, bad;                                                       // no action has any probability; a NaN or plus infinity is among them
    __device__ __forceinline__ Known(const Part& p) {
        nothing = p.s == 0.0f; bad = !(p.s == p.s);
        m = p.m; log2_s = log2f(p.s); h = nothing ? 0.0f : LN2 * (log2_s - p.t / p.s);
    }
    // Log probability of an action with this logit.
    __device__ __forceinline__ float logprob(float x, const Rows& p) const {
        if (bad) return log2_s;
        if (x == NONE || nothing) return NONE;
        const float c = p.scale * LOG2E;
        if (!(fabsf(x) < LARGE && is_usual(m, c))) return (x - m) * p.scale - LN2 * log2_s;
        return LN2 * (fmaf(x, c, -(m * c)) - log2_s);
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
    static __device__ __forceinline__ uint4 fill() { const unsigned f = __float_as_uint(FLOOR); return make_uint4(f, f, f, f); }
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
    static __device__ __forceinline__ uint4 fill() { return make_uint4(FLOOR2, FLOOR2, FLOOR2, FLOOR2); }
    static __device__ __forceinline__ unsigned up(unsigned v) { unsigned r; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(FLOOR2)); return r; }
    static __device__ __forceinline__ void floored(const uint4& v, float (&x)[8]) { values(make_uint4(up(v.x), up(v.y), up(v.z), up(v.w)), x); }
    static __device__ __forceinline__ unsigned two16(float a, float b) { const __nv_bfloat162 v = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const unsigned*>(&v); }
    static __device__ __forceinline__ uint4 pack(const float (&x)[8]) { return make_uint4(two16(x[0], x[1]), two16(x[2], x[3]), two16(x[4], x[5]), two16(x[6], x[7])); }
};
template <> struct Chunk<CUDARL_F16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void pair(unsigned v, float& a, float& b) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v)); a = f.x; b = f.y; }
    static __device__ __forceinline__ void values(const uint4& v, float (&x)[8]) { pair(v.x, x[0], x[1]); pair(v.y, x[2], x[3]); pair(v.z, x[4], x[5]); pair(v.w, x[6], x[7]); }
    static __device__ __forceinline__ uint4 fill() { return make_uint4(0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u, 0xFC00FC00u); }      // minus infinity: FLOOR is not an f16
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

// ------------------------------------------------------------------------------------------------------------------ short rows
// G lanes a row, E values a lane in registers: up to G E actions.  The sums of a row need log2(G) exchanges; every load of a lane is one 16- or 32-byte
// piece where rows are aligned to it.
template <int TYPE, int E>
__device__ __forceinline__ void load_short(const Rows& p, long long r, int j0, bool wide, float (&x)[E]) {
    using O = Of<TYPE>;
    const auto* at = static_cast<const typename O::T*>(p.logits) + r * p.stride + j0;
    if (wide && j0 + E <= p.actions) {
        constexpr int BYTES = E * (int)sizeof(typename O::T);
        if constexpr (BYTES == 8) {
            const uint2 v = *reinterpret_cast<const uint2*>(at);
            Chunk<TYPE>::pair(v.x, x[0], x[1]); Chunk<TYPE>::pair(v.y, x[2], x[3]);
        } else {
#pragma unroll
            for (int k = 0; k < BYTES / 16; ++k) {
                float part[Chunk<TYPE>::N];
                Chunk<TYPE>::values(reinterpret_cast<const uint4*>(at)[k], part);
#pragma unroll
                for (int i = 0; i < Chunk<TYPE>::N; ++i) x[k * Chunk<TYPE>::N + i] = part[i];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = j0 + i < p.actions ? O::get(at[i]) : NONE;
    }
}
template <int E>
__device__ __forceinline__ void mask_short(const Rows& p, long long r, int j0, unsigned& bits) {
    const unsigned char* legal = p.legal + r * p.legal_stride + j0;
    bits = 0u;
#pragma unroll
    for (int i = 0; i < E; ++i) bits |= j0 + i < p.actions && __ldg(legal + i) ? 1u << i : 0u;
}

template <int TYPE, int G, int E, bool TOP>
__global__ void __launch_bounds__(256) k_short(Rows p, Outputs o, bool wide) {
    const int lane = (int)threadIdx.x % G, j0 = lane * E;
    const long long step = (long long)gridDim.x * (256 / G);
    // (the loop is the same for all lanes of a warp: rows behind the last are computed from the last and not written)
    for (long long first = (long long)blockIdx.x * (256 / G); first < p.rows; first += step) {
        const long long mine = first + (int)threadIdx.x / G, r = mine < p.rows ? mine : p.rows - 1;
        const bool write = mine < p.rows;
        float x[E];
        load_short<TYPE, E>(p, r, j0, wide, x);
        if (p.legal) {
            unsigned bits;
            mask_short<E>(p, r, j0, bits);
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = bits >> i & 1u ? x[i] : NONE;
        }
        const int a = p.taken ? __ldg(p.taken + r) : -1;
        float m = x[0];
#pragma unroll
        for (int i = 1; i < E; ++i) m = fmaxf(m, x[i]);
#pragma unroll
        for (int by = 1; by < G; by *= 2) m = fmaxf(m, __shfl_xor_sync(ALL, m, by));
        const float c = p.scale * LOG2E, mc = m * c, from = m == NONE ? 0.0f : m;
        const bool exact = !is_usual(m, c);
        Part part{m, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < E; ++i) {
            float y = fmaf(max_nan(x[i], FLOOR), c, -mc);
            if (exact) y = (x[i] - from) * p.scale * LOG2E;
            const float e = exp2_fast(y);
            part.s += e;
            part.t += e > 0.0f ? y * e : 0.0f;
        }
#pragma unroll
        for (int by = 1; by < G; by *= 2) { part.s += __shfl_xor_sync(ALL, part.s, by); part.t += __shfl_xor_sync(ALL, part.t, by); }
        const Known known(part);
        if (write) {
            if (lane == 0) known.write(o, r);
            if (o.logprob) {
                if ((unsigned)a >= (unsigned)p.actions) { if (lane == 0) o.logprob[r] = known.bad ? known.log2_s : 0.0f; }
                else if ((unsigned)(a - j0) < (unsigned)E) {                 // the lane that holds it
                    float xa = x[0];
#pragma unroll
                    for (int i = 1; i < E; ++i) xa = a - j0 == i ? x[i] : xa;
                    o.logprob[r] = known.logprob(xa, p);
                }
            }
        }
        if constexpr (TOP) {
            // every lane's own values in falling order, then the largest head of the G lists, `top` times
            unsigned long long key[E];
#pragma unroll
            for (int i = 0; i < E; ++i) key[i] = x[i] > NONE && !known.bad ? order_key(x[i], (unsigned)(j0 + i)) : 0ull;
#pragma unroll
            for (int size = 2; size <= E; size *= 2)
#pragma unroll
                for (int by = size / 2; by; by /= 2)
#pragma unroll
                    for (int i = 0; i < E; ++i)
                        if ((i & by) == 0) {
                            const bool falling = (i & size) == 0 || size == E;
                            const unsigned long long u = key[i], v = key[i | by];
                            const bool swap = falling ? u < v : u > v;
                            key[i] = swap ? v : u; key[i | by] = swap ? u : v;
                        }
            for (int k = 0; k < o.top; ++k) {
                unsigned long long best = key[0];
#pragma unroll
                for (int by = 1; by < G; by *= 2) { const unsigned long long other = __shfl_xor_sync(ALL, best, by); best = best > other ? best : other; }
                if (best == 0ull ? lane == 0 : key[0] == best) {
                    if (write) {
                        o.top_actions[r * o.top + k] = best ? key_action(best) : -1;
                        o.top_logprobs[r * o.top + k] = known.bad ? known.log2_s : best ? known.logprob(key_value(best), p) : NONE;
                    }
#pragma unroll
                    for (int i = 0; i + 1 < E; ++i) key[i] = key[i + 1];
                    key[E - 1] = 0ull;
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------ long rows
// T threads a row (a warp, or a block), or the blocks of a cluster for few rows.  A thread takes batches of UNROLL chunks; a batch costs one maximum and one
// rebasing of the thread's sums.  The threads' parts are joined by shuffles, in shared memory, and over the cluster in the other blocks' shared memory.
//
// Alternatives: the maximum of every batch (of every GROUP of batches, for very long rows) is kept in shared memory.  With W warps in all, the ceil(top / W)-th
// largest thread maximum of each warp, and of those the least, is a bound that at least `top` values of the row reach.  Only batches that reach it are read
// again -- a few dozen of them -- and what reaches the bound there is put in order by one warp.  Where too much does (rows of equal values) or too little (fewer
// than `top` values above FLOOR), every value of the row is gone through again, each warp with its 32 best in registers.
constexpr int UNROLL = 4, TABLE_ROWS = 32, LIST = 192, CANDIDATES = 256;

template <int T> struct Shared {
    Part part[T / 32];
    Part block;                          // of this block, for the other blocks of the cluster
    float bound[T / 32];
    float block_bound;
    unsigned listed, found;
    unsigned list[LIST];
    unsigned long long key[CANDIDATES];
};

template <int T> __device__ __forceinline__ void team_sync() { if constexpr (T == 32) __syncwarp(); else __syncthreads(); }

template <int TYPE, int T, bool MASKED, bool TOP>
__global__ void __launch_bounds__(T == 32 ? 128 : T, T == 32 ? 6 : 4) k_long(Rows p, Outputs o, int blocks, int group) {
    using C = Chunk<TYPE>;
    using Value = typename Of<TYPE>::T;
    constexpr int N = C::N, TEAMS = T == 32 ? 4 : 1, WARPS = T / 32;
    extern __shared__ __align__(16) unsigned char shared_bytes[];
    __shared__ Shared<T> shared_all[TEAMS];
    const int team = T == 32 ? (int)threadIdx.x / 32 : 0, t = (int)threadIdx.x % T, warp = t / 32;
    const unsigned lane = threadIdx.x % 32u;
    Shared<T>& sh = shared_all[team];
    Value* table = reinterpret_cast<Value*>(shared_bytes) + team * (TABLE_ROWS + 1) * T;
    const int rank = blocks > 1 ? (int)(blockIdx.x % (unsigned)blocks) : 0, threads = blocks * T, me = rank * T + t;
    const float c = p.scale * LOG2E;
    const long long first = (long long)(blockIdx.x / (unsigned)blocks) * TEAMS + team, step = (long long)(gridDim.x / (unsigned)blocks) * TEAMS;
    for (long long r = first; r < p.rows; r += step) {
        const Row<TYPE> row(p, r);
        const int batches = (row.chunks + UNROLL * threads - 1) / (UNROLL * threads);
        const int a = t == 0 && rank == 0 && p.taken ? __ldg(p.taken + r) : -1;
        Part part{FLOOR, 0.0f, 0.0f};
        Two s2 = two(0.0f, 0.0f), t2 = s2;
        float high = FLOOR;                                                  // of the group of batches
        for (int b = 0; b < batches; ++b) {
            uint4 raw[UNROLL];
            unsigned legal[UNROLL][N / 4];
            const int at = b * UNROLL * threads + me;
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int k = at + u * threads;
                raw[u] = k < row.chunks ? row.chunk(k) : C::fill();
                if constexpr (MASKED) {
                    if (k < row.chunks) mask_words<N>(row.legal, row.head + k * N, row.actions, legal[u]);
                    else
#pragma unroll
                        for (int i = 0; i < N / 4; ++i) legal[u][i] = 0u;
                }
            }
            float x[UNROLL][N], bm = FLOOR;
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                C::floored(raw[u], x[u]);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if constexpr (MASKED) x[u][i] = is_legal<N>(legal[u], i) ? x[u][i] : FLOOR;
                    bm = fmaxf(bm, x[u][i]);
                }
            }
            if constexpr (TOP) {
                high = fmaxf(high, bm);
                if ((b + 1) % group == 0 || b + 1 == batches) { table[(b / group) * T + t] = Of<TYPE>::put(high); high = FLOOR; }
            }
            if (bm > part.m) {
                float u, v;
                apart(s2, u, v); part.s += u + v; apart(t2, u, v); part.t += u + v;
                s2 = two(0.0f, 0.0f); t2 = s2;
                rebase(part, bm, c);
            }
            const Two c2 = two(c, c), mc2 = two(-base_of(part.m, c), -base_of(part.m, c));
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
#pragma unroll
                for (int i = 0; i < N; i += 2) {
                    const Two y2 = fma2(two(x[u][i], x[u][i + 1]), c2, mc2);
                    float y0, y1;
                    apart(y2, y0, y1);
                    const Two e2 = two(exp2_fast(y0), exp2_fast(y1));
                    s2 = add2(s2, e2);
                    t2 = fma2(y2, e2, t2);
                }
        }
        { float u, v; apart(s2, u, v); part.s += u + v; apart(t2, u, v); part.t += u + v; }
        const bool has_end = me < row.ends;                                  // (ends < 2 N <= 32 <= T: all in the first block)
        const float xe = has_end ? max_nan(row.at(row.end(me)), FLOOR) : FLOOR;
        if (has_end) take_one(part, xe, c);
        if constexpr (TOP) table[TABLE_ROWS * T + t] = Of<TYPE>::put(xe == xe ? xe : FLOOR);
        const float own = part.m;                                            // this thread's maximum

        // join
#pragma unroll
        for (int by = 16; by; by /= 2) {
            Part other;
            other.m = __shfl_xor_sync(ALL, part.m, by); other.s = __shfl_xor_sync(ALL, part.s, by); other.t = __shfl_xor_sync(ALL, part.t, by);
            join(part, other, c);
        }
        if constexpr (TOP) {                                                 // the warp's part of the bound
            const int rank_wanted = (o.top + WARPS * blocks - 1) / (WARPS * blocks);
            unsigned b = __float_as_uint(own);
            b = (b & 0x80000000u) ? ~b : b | 0x80000000u;
            unsigned high_bits = 0u;
            for (int k = 0; k < rank_wanted; ++k) {
                high_bits = __reduce_max_sync(ALL, b);
                const unsigned holders = __ballot_sync(ALL, b == high_bits);
                if (lane == (unsigned)__ffs((int)holders) - 1u) b = 0u;
            }
            if (lane == 0) sh.bound[warp] = high_bits == 0u ? FLOOR : __uint_as_float((high_bits & 0x80000000u) ? high_bits & 0x7FFFFFFFu : ~high_bits);
            if (t == 0) sh.listed = sh.found = 0u;
        }
        if constexpr (T > 32) {
            if (lane == 0) sh.part[warp] = part;
            __syncthreads();
            part = sh.part[0];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) join(part, sh.part[w], c);
        } else __syncwarp();
        float bound = FLOOR;
        if constexpr (TOP) {
            bound = sh.bound[0];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) bound = fminf(bound, sh.bound[w]);
        }
        if constexpr (T > 32) {
            if (blocks > 1) {
                if (t == 0) { sh.block = part; sh.block_bound = bound; }
                cg::cluster_group cluster = cg::this_cluster();
                cluster.sync();
                part = cluster.map_shared_rank(&sh, 0)->block;
                for (int k = 1; k < blocks; ++k) join(part, cluster.map_shared_rank(&sh, k)->block, c);
                if constexpr (TOP)
                    for (int k = 0; k < blocks; ++k) bound = fminf(bound, cluster.map_shared_rank(&sh, k)->block_bound);
            }
        }
        if (!is_usual(part.m, c)) {
            // beyond the limit: the maximum itself, then sums of exact differences; every block of a cluster goes through the whole row
            float m = NONE;
            for (int j = t; j < row.actions; j += T) m = fmaxf(m, row.at(j));
#pragma unroll
            for (int by = 16; by; by /= 2) m = fmaxf(m, __shfl_xor_sync(ALL, m, by));
            if constexpr (T > 32) {
                __syncthreads();
                if (lane == 0) sh.part[warp].m = m;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < WARPS; ++w) m = fmaxf(m, sh.part[w].m);
            }
            const float from = m == NONE ? 0.0f : m;
            float s = 0.0f, sum = 0.0f;
            for (int j = t; j < row.actions; j += T) {
                const float y = (row.at(j) - from) * p.scale * LOG2E, e = exp2_fast(y);
                s += e;
                sum += e > 0.0f ? y * e : 0.0f;
            }
#pragma unroll
            for (int by = 16; by; by /= 2) { s += __shfl_xor_sync(ALL, s, by); sum += __shfl_xor_sync(ALL, sum, by); }
            part = Part{m, s, sum};
            if constexpr (T > 32) {
                if (lane == 0) { sh.part[warp].s = s; sh.part[warp].t = sum; }
                __syncthreads();
                part.s = part.t = 0.0f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) { part.s += sh.part[w].s; part.t += sh.part[w].t; }
            }
        }
        const Known known(part);
        if (t == 0 && rank == 0) {
            known.write(o, r);
            if (o.logprob) o.logprob[r] = known.bad ? known.log2_s : (unsigned)a >= (unsigned)row.actions ? 0.0f : known.logprob(row.at(a), p);
        }
        if constexpr (TOP) {
            // batches that reach the bound, then what reaches it in them
            const int rows_used = (batches + group - 1) / group;
            auto list_it = [&](int q) {
                const unsigned place = atomicAdd(&sh.listed, 1u);
                if (place < LIST) sh.list[place] = (unsigned)(q * T + t);
            };
            if (bound > ABOVE_FLOOR && own >= bound) {
                for (int q = 0; q < rows_used; ++q)
                    if (Of<TYPE>::get(table[q * T + t]) >= bound) list_it(q);
                if (xe >= bound) list_it(TABLE_ROWS);
            }
            team_sync<T>();
            const unsigned listed = min(sh.listed, (unsigned)LIST);
            for (unsigned l = (unsigned)warp; l < listed; l += WARPS) {
                const int q = (int)sh.list[l] / T, owner = rank * T + (int)sh.list[l] % T;
                const int values = q == TABLE_ROWS ? 1 : group * UNROLL * N;
                for (int e = (int)lane; e < values; e += 32) {
                    int j = -1;
                    if (q == TABLE_ROWS) j = row.end(owner);
                    else {
                        const int k = (q * group * UNROLL + e / N) * threads + owner;
                        if (k < row.chunks) j = row.head + k * N + e % N;
                    }
                    const float x = j >= 0 ? row.at(j) : NONE;
                    if (x >= bound) {
                        const unsigned place = atomicAdd(&sh.found, 1u);
                        if (place < CANDIDATES) sh.key[place] = order_key(x, (unsigned)j);
                    }
                }
            }
            if (T > 32 && blocks > 1) cg::this_cluster().sync(); else team_sync<T>();
            if (rank == 0) {
                unsigned total = 0u;
                bool over = !(bound > ABOVE_FLOOR);
                for (int k = 0; k < blocks; ++k) {
                    const Shared<T>* from = &sh;
                    if constexpr (T > 32) if (blocks > 1) from = cg::this_cluster().map_shared_rank(&sh, k);
                    total += from->found;
                    over = over || from->listed > (unsigned)LIST || from->found > (unsigned)CANDIDATES;
                }
                over = over || total < (unsigned)o.top;
                unsigned long long best = 0ull;
                if (known.bad || known.nothing) {}
                else if (!over) {
                    if (warp == 0)
                        for (int k = 0; k < blocks; ++k) {
                            const Shared<T>* from = &sh;
                            if constexpr (T > 32) if (blocks > 1) from = cg::this_cluster().map_shared_rank(&sh, k);
                            const unsigned n = from->found;
                            for (unsigned l = 0; l < n; l += 32u) take32(best, l + lane < n ? from->key[l + lane] : 0ull, lane, o.top);
                        }
                } else {
                    for (int j0 = warp * 32; j0 < row.actions; j0 += T) {
                        const int j = j0 + (int)lane;
                        const float x = j < row.actions ? row.at(j) : NONE;
                        take32(best, x > NONE ? order_key(x, (unsigned)j) : 0ull, lane, o.top);
                    }
                    if constexpr (T > 32) {
                        __syncthreads();                                     // the keys of the short way have been counted by all
                        if (WARPS * 32 <= CANDIDATES) sh.key[warp * 32 + lane] = best;
                        __syncthreads();
                        if (warp == 0)
                            for (int w = 1; w < WARPS; ++w) best = merged32(best, sh.key[w * 32 + lane], lane);
                    }
                }
                if (warp == 0 && (int)lane < o.top) {
                    o.top_actions[r * o.top + lane] = best ? key_action(best) : -1;
                    o.top_logprobs[r * o.top + lane] = known.bad ? known.log2_s : best ? known.logprob(key_value(best), p) : NONE;
                }
            }
        }
        if (T > 32 && blocks > 1) cg::this_cluster().sync();                 // nobody leaves, or begins the next row, while its shared memory is read
        else if constexpr (T > 32 || TOP) team_sync<T>();
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

template <int TYPE, int G, int E>
__global__ void __launch_bounds__(256) k_short_backward(Rows p, const float4* stats, const float* grad_logprob, const float* grad_entropy, void* grad, long long grad_stride, bool wide,
                                                        bool wide_grad) {
    using O = Of<TYPE>;
    const int lane = (int)threadIdx.x % G, j0 = lane * E;
    const long long step = (long long)gridDim.x * (256 / G);
    for (long long r = (long long)blockIdx.x * (256 / G) + (int)threadIdx.x / G; r < p.rows; r += step) {
        float x[E];
        load_short<TYPE, E>(p, r, j0, wide, x);
        const Slope slope(p, stats, grad_logprob, grad_entropy, r);
        unsigned bits = ~0u;
        if (p.legal) mask_short<E>(p, r, j0, bits);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = bits >> i & 1u ? slope.one(x[i], j0 + i) : 0.0f;
        auto* at = static_cast<typename O::T*>(grad) + r * grad_stride + j0;
        if (wide_grad && j0 + E <= p.actions) {
            constexpr int BYTES = E * (int)sizeof(typename O::T);
            if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(at) = make_uint2(Chunk<TYPE>::two16(x[0], x[1]), Chunk<TYPE>::two16(x[2], x[3]));
            else
#pragma unroll
                for (int k = 0; k < BYTES / 16; ++k) {
                    float part[Chunk<TYPE>::N];
#pragma unroll
                    for (int i = 0; i < Chunk<TYPE>::N; ++i) part[i] = x[k * Chunk<TYPE>::N + i];
                    reinterpret_cast<uint4*>(at)[k] = Chunk<TYPE>::pack(part);
                }
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) if (j0 + i < p.actions) at[i] = O::put(x[i]);
        }
    }
}

// Long rows: T threads take UNROLL chunks each of a piece of a row; chunks begin where the gradient's address is aligned, and the logits are read in the same
// chunks where their address is too, else one by one.
template <int TYPE, int T, bool MASKED>
__global__ void __launch_bounds__(256) k_long_backward(Rows p, const float4* stats, const float* grad_logprob, const float* grad_entropy, void* grad, long long grad_stride, int pieces) {
    using C = Chunk<TYPE>;
    using O = Of<TYPE>;
    constexpr int N = C::N, TEAMS = 256 / T;
    const int team = (int)threadIdx.x / T, t = (int)threadIdx.x % T;
    const long long work = p.rows * pieces, step = (long long)gridDim.x * TEAMS;
    for (long long w = (long long)blockIdx.x * TEAMS + team; w < work; w += step) {
        const long long r = pieces == 1 ? w : w / pieces;
        const int piece = pieces == 1 ? 0 : (int)(w - r * pieces);
        const auto* x = static_cast<const typename O::T*>(p.logits) + r * p.stride;
        auto* g = static_cast<typename O::T*>(grad) + r * grad_stride;
        const unsigned char* legal = MASKED ? p.legal + r * p.legal_stride : nullptr;
        const int head = min((int)((16u - ((unsigned)reinterpret_cast<uintptr_t>(g) & 15u)) & 15u) / (int)sizeof(typename O::T), p.actions);
        const int chunks = (p.actions - head) / N, ends = p.actions - chunks * N;
        const bool together = (((unsigned)reinterpret_cast<uintptr_t>(x) ^ (unsigned)reinterpret_cast<uintptr_t>(g)) & 15u) == 0u;
        const Slope slope(p, stats, grad_logprob, grad_entropy, r);
        if (piece == 0 && t < ends) {
            const int j = t < head ? t : chunks * N + t;
            g[j] = O::put(MASKED && !__ldg(legal + j) ? 0.0f : slope.one(O::get(x[j]), j));
        }
        const bool usual = slope.usual();
        const Two c2 = two(slope.c, slope.c), mc2 = two(-slope.mc, -slope.mc), l2 = two(-slope.log2_s, -slope.log2_s), A2 = two(slope.A, slope.A), B2 = two(slope.B, slope.B),
                  minus = two(-1.0f, -1.0f);
        for (int base = piece * UNROLL * T; base < chunks; base += pieces * UNROLL * T) {
            uint4 raw[UNROLL];
            unsigned mask[UNROLL][N / 4];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int k = base + u * T + t;
                raw[u] = C::fill();
                if (k < chunks) {
                    const auto* at = x + head + k * N;
                    if (together) raw[u] = *reinterpret_cast<const uint4*>(at);
                    else raw[u] = gather_chunk(at);
                    if constexpr (MASKED) mask_words<N>(legal, head + k * N, p.actions, mask[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int k = base + u * T + t;
                if (k >= chunks) continue;
                float v[N];
                const int j0 = head + k * N;
                if (usual && (unsigned)(slope.taken - j0) >= (unsigned)N) {
                    C::floored(raw[u], v);
#pragma unroll
                    for (int i = 0; i < N; i += 2) {
                        const Two lp2 = add2(fma2(two(v[i], v[i + 1]), c2, mc2), l2);
                        float a, b;
                        apart(lp2, a, b);
                        apart(mul2(mul2(two(exp2_fast(a), exp2_fast(b)), minus), fma2(B2, lp2, A2)), v[i], v[i + 1]);
                    }
                } else {
                    C::values(raw[u], v);
#pragma unroll
                    for (int i = 0; i < N; ++i) v[i] = slope.one(v[i], j0 + i);
                }
                if constexpr (MASKED)
#pragma unroll
                    for (int i = 0; i < N; ++i) v[i] = is_legal<N>(mask[u], i) ? v[i] : 0.0f;
                *reinterpret_cast<uint4*>(g + j0) = C::pack(v);
            }
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

constexpr int SHORT_ACTIONS = 128, WARP_ACTIONS = 2048;

template <int TYPE, int G, int E>
cudaError_t launch_short(const Rows& p, const Outputs& o, cudaStream_t st) {
    constexpr int value = (int)sizeof(typename Of<TYPE>::T), bytes = E * value < 16 ? E * value : 16;
    const bool wide = aligned_rows(p.logits, p.stride, value, bytes);
    const unsigned grid = blocks_of(p.rows, 256 / G);
    if (o.top) k_short<TYPE, G, E, true><<<grid, 256, 0, st>>>(p, o, wide);
    else k_short<TYPE, G, E, false><<<grid, 256, 0, st>>>(p, o, wide);
    return cudaGetLastError();
}

template <int TYPE, int T, bool MASKED, bool TOP>
cudaError_t launch_long(const Rows& p, const Outputs& o, int blocks, cudaStream_t st) {
    constexpr int TEAMS = T == 32 ? 4 : 1, N = Chunk<TYPE>::N;
    const long long batches = ((long long)p.actions / N + UNROLL * (long long)T * blocks - 1) / (UNROLL * (long long)T * blocks);
    const int group = (int)((batches + TABLE_ROWS - 1) / TABLE_ROWS > 1 ? (batches + TABLE_ROWS - 1) / TABLE_ROWS : 1);
    const size_t table = TOP ? (size_t)(TABLE_ROWS + 1) * T * TEAMS * sizeof(typename Of<TYPE>::T) : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(T == 32 ? 128 : T);
    cfg.dynamicSmemBytes = table;
    cfg.stream = st;
    const unsigned teams = blocks_of(p.rows, TEAMS);
    cfg.gridDim = dim3((teams < 1u << 24 ? teams : 1u << 24) * (unsigned)blocks);
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
    const int v = p.actions;
    if (v <= 4) return launch_short<TYPE, 1, 4>(p, o, st);
    if (v <= 8) return launch_short<TYPE, 1, 8>(p, o, st);
    if (v <= 16) return launch_short<TYPE, 2, 8>(p, o, st);
    if (v <= 32) return launch_short<TYPE, 4, 8>(p, o, st);
    if (v <= 64) return launch_short<TYPE, 8, 8>(p, o, st);
    if (v <= SHORT_ACTIONS) return launch_short<TYPE, 16, 8>(p, o, st);
    if (v <= WARP_ACTIONS) return launch_long<TYPE, 32>(p, o, 1, st);
    // a cluster for each row where there are too few rows to occupy the GPU, as long as each block still gets half a batch
    int blocks = 1;
    while (blocks < 8 && p.rows * blocks * 2 <= sms * 2 && (long long)v >= 256ll * Chunk<TYPE>::N * UNROLL / 2 * blocks * 2) blocks *= 2;
    return launch_long<TYPE, 256>(p, o, blocks, st);
}

struct BackwardArgs { const float4* stats; const float* gl; const float* gh; void* grad; long long stride; };

template <int TYPE, int G, int E>
cudaError_t launch_short_backward(const Rows& p, const BackwardArgs& b, cudaStream_t st) {
    constexpr int value = (int)sizeof(typename Of<TYPE>::T), bytes = E * value < 16 ? E * value : 16;
    k_short_backward<TYPE, G, E><<<blocks_of(p.rows, 256 / G), 256, 0, st>>>(p, b.stats, b.gl, b.gh, b.grad, b.stride, aligned_rows(p.logits, p.stride, value, bytes),
                                                                             aligned_rows(b.grad, b.stride, value, bytes));
    return cudaGetLastError();
}
template <int TYPE, int T>
cudaError_t launch_long_backward(const Rows& p, const BackwardArgs& b, cudaStream_t st) {
    const long long each = (long long)T * UNROLL * Chunk<TYPE>::N;
    const int pieces = T == 32 ? 1 : (int)((p.actions + each - 1) / each);
    const unsigned grid = p.rows > (1ll << 50) / pieces ? 1u << 28 : blocks_of(p.rows * pieces, 256 / T);
    if (p.legal) k_long_backward<TYPE, T, true><<<grid, 256, 0, st>>>(p, b.stats, b.gl, b.gh, b.grad, b.stride, pieces);
    else k_long_backward<TYPE, T, false><<<grid, 256, 0, st>>>(p, b.stats, b.gl, b.gh, b.grad, b.stride, pieces);
    return cudaGetLastError();
}
template <int TYPE>
cudaError_t launch_backward(const Rows& p, const BackwardArgs& b, cudaStream_t st) {
    const int v = p.actions;
    if (v <= 4) return launch_short_backward<TYPE, 1, 4>(p, b, st);
    if (v <= 8) return launch_short_backward<TYPE, 1, 8>(p, b, st);
    if (v <= 16) return launch_short_backward<TYPE, 2, 8>(p, b, st);
    if (v <= 32) return launch_short_backward<TYPE, 4, 8>(p, b, st);
    if (v <= 64) return launch_short_backward<TYPE, 8, 8>(p, b, st);
    if (v <= SHORT_ACTIONS) return launch_short_backward<TYPE, 16, 8>(p, b, st);
    if (v <= WARP_ACTIONS) return launch_long_backward<TYPE, 32>(p, b, st);
    return launch_long_backward<TYPE, 256>(p, b, st);
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
        (rc = arrays.check("stats", stats, 16)) || (rc = arrays.check_if("grad_logprob", grad_logprob, 4)) || (rc = arrays.check_if("grad_entropy", grad_entropy, 4)) ||
        (rc = arrays.check("grad_logits", grad_logits, align))) return rc;
    CurrentDevice current;
    cudaError_t e = current.set(arrays.device());
    if (e != cudaSuccess) return fail_cuda("cudaSetDevice", e);
    const Rows r = device_rows(p);
    const BackwardArgs b{reinterpret_cast<const float4*>(stats), grad_logprob, grad_entropy, grad_logits, (long long)grad_stride};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    e = p->type == CUDARL_F32 ? launch_backward<CUDARL_F32>(r, b, st) : p->type == CUDARL_BF16 ? launch_backward<CUDARL_BF16>(r, b, st) : launch_backward<CUDARL_F16>(r, b, st);
    return e == cudaSuccess ? 0 : fail_cuda("cudarl_policy_logprobs_backward", e);
}
