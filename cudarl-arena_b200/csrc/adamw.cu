// adamw.cu -- one AdamW step over all tensors of a network, moments in 32 bits or in 8, with clipping by the global norm.
//
// The handle keeps on the device: the list of the tensors, a list of the pieces of them that a block of threads takes at a time (up to eight blocks of 256 values,
// a block being what one scale of the 8-bit moments is for), and the step count with what depends on it.  Nothing of a step comes from the host but lr and grad_scale, so a
// captured step counts on.
//
// What bounds it (B200, kernels alone): with 32-bit moments the memory: 150M values of bf16 weights with masters, 28 bytes each, 695 us = 6.05 TB/s, 92 % of a copy's rate.
// With 8-bit moments, 16 bytes a value, neither the memory (40M values 137 us: 640 MB in and out = 4.7 TB/s, 585 MB of them past the L2) nor the issue slots (590
// instructions for a warp's 256 values, 0.60 issued per scheduler and cycle): the warps of a block have their arithmetic at the same time -- for each issue 1.7 warps
// that could have issued too and 1.3 that wait for an occupied unit -- and then wait for their pieces together.  200M with the norm 740 - 785 us, by the box.
#include "async_copy.cuh"
#include "caller_arrays.cuh"
#include "rules.cuh"
#include <cuda_fp8.h>
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

namespace {
using namespace cudarl;

constexpr unsigned TAG_OPTIMIZER = 0x4F50544Du;
constexpr int BLOCK = CUDARL_ADAMW_BLOCK;
constexpr int WARPS = 8, THREADS = 32 * (WARPS + 1);     // eight warps that compute, and one that has their next pieces copied
constexpr int RESIDENT = 3;                    // blocks of threads on an SM

struct Tensor {
    void* param; const void* grad; float* master; void* moment1; void* moment2; float* scale1; float* scale2;
    long long count;
    float lr_scale, decay;
    unsigned char param_type, grad_type;
    unsigned char wide;                       // every array but the gradient begins at an address that bulk copies can start at and eight values can be stored to at once
    unsigned char copied_grad;                // bulk copies of the gradient can start where it begins (16 bytes) ...
    unsigned char wide_grad;                  // ... and eight of its values can be loaded at once (32 bytes for those of 32 bits)
};
struct Piece { unsigned tensor, block, blocks, number; };   // `blocks` blocks (1 .. WARPS) of a tensor from its block `block` on, which is number `number` of all

struct Control {
    long long step, skipped;
    double norm, power1, power2;              // powers of the betas for the step to come ...
    float fix1, root_fix2;                    // ... and what they make of it: 1 / (1 - power1), and the root of 1 / (1 - power2).  fix1 is 0 once a wait has run out
    float clip;
    unsigned go;                              // 0: the norm was no finite number
    unsigned done, done_norm;                 // blocks of the launch that have finished
    unsigned error;                           // CUDARL_DEVERR_*
};

struct Settings {
    float beta1, rest1, beta2, rest2, eps;    // rest = 1 - beta
    float one;                                // 1
    unsigned keys[20];                        // of the ten Philox rounds
    int clipped;
    unsigned polls;                           // > 0: of a test, see cudarl_debug_adamw_set_copy_wait_polls
    double power1, power2;                    // the betas
};

// Eight values from `i` on as they lie there: one access of 16 or 32 bytes where `wide`, else one by one up to `len` (zeros behind that).  They are made
// floats of in a call of its own, so that a thread has all its loads on their way before it waits for the first.
struct Raw { unsigned v[8]; };
__device__ __forceinline__ void load8(Raw& r, const void* p, int type, long long i, bool wide, int len) {
    if (type == CUDARL_F32) {
        const unsigned* at = static_cast<const unsigned*>(p) + i;
        if (wide) asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : "=r"(r.v[0]), "=r"(r.v[1]), "=r"(r.v[2]), "=r"(r.v[3]), "=r"(r.v[4]), "=r"(r.v[5]), "=r"(r.v[6]), "=r"(r.v[7]) : "l"(at));
        else {
#pragma unroll
            for (int k = 0; k < 8; ++k) r.v[k] = k < len ? at[k] : 0u;
        }
    } else {
        const unsigned short* at = static_cast<const unsigned short*>(p) + i;
        if (wide) asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.v[0]), "=r"(r.v[1]), "=r"(r.v[2]), "=r"(r.v[3]) : "l"(at));
        else {
#pragma unroll
            for (int k = 0; k < 4; ++k) r.v[k] = (2 * k < len ? at[2 * k] : 0u) | (2 * k + 1 < len ? (unsigned)at[2 * k + 1] << 16 : 0u);
        }
    }
}
__device__ __forceinline__ void floats8(const Raw& r, int type, float (&x)[8]) {
    if (type == CUDARL_F32) {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = __uint_as_float(r.v[k]);
    }
    else if (type == CUDARL_BF16) {
#pragma unroll
        for (int k = 0; k < 4; ++k) { x[2 * k] = __uint_as_float(r.v[k] << 16); x[2 * k + 1] = __uint_as_float(r.v[k] & 0xFFFF0000u); }
    }
    else {
#pragma unroll
        for (int k = 0; k < 4; ++k) { const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.v[k])); x[2 * k] = f.x; x[2 * k + 1] = f.y; }
    }
}
__device__ __forceinline__ void store8(void* p, int type, long long i, bool wide, int len, const float (&x)[8]) {
    if (type == CUDARL_F32) {
        float* at = static_cast<float*>(p) + i;
        if (wide) asm volatile("st.global.v8.f32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" :: "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]), "l"(at) : "memory");
        else {
#pragma unroll
            for (int k = 0; k < 8; ++k) if (k < len) at[k] = x[k];
        }
        return;
    }
    unsigned v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (type == CUDARL_BF16) { const __nv_bfloat162 w = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]); v[k] = *reinterpret_cast<const unsigned*>(&w); }
        else { const __half2 w = __floats2half2_rn(x[2 * k], x[2 * k + 1]); v[k] = *reinterpret_cast<const unsigned*>(&w); }
    }
    if (wide) *reinterpret_cast<uint4*>(static_cast<unsigned short*>(p) + i) = make_uint4(v[0], v[1], v[2], v[3]);
    else {
        unsigned short* at = static_cast<unsigned short*>(p) + i;
#pragma unroll
        for (int k = 0; k < 8; ++k) if (k < len) at[k] = (unsigned short)(v[k / 2] >> (k % 2 ? 16 : 0));
    }
}
__device__ __forceinline__ uint2 load_codes(const void* p, long long i, bool wide, int len) {
    const unsigned char* at = static_cast<const unsigned char*>(p) + i;
    if (wide) return *reinterpret_cast<const uint2*>(at);
    unsigned v[2] = {0u, 0u};
#pragma unroll
    for (int k = 0; k < 8; ++k) if (k < len) v[k / 4] |= (unsigned)at[k] << (8 * (k % 4));
    return make_uint2(v[0], v[1]);
}
__device__ __forceinline__ void store_codes(void* p, long long i, bool wide, int len, uint2 c) {
    unsigned char* at = static_cast<unsigned char*>(p) + i;
    if (wide) { *reinterpret_cast<uint2*>(at) = c; return; }
#pragma unroll
    for (int k = 0; k < 8; ++k) if (k < len) at[k] = (unsigned char)((k < 4 ? c.x : c.y) >> (8 * (k % 4)));
}
__device__ __forceinline__ void from_codes(unsigned v, float* x) {           // four codes
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(v >> (16 * k)), __NV_E4M3));
        const float2 f = __half22float2(h);
        x[2 * k] = f.x; x[2 * k + 1] = f.y;
    }
}

// Whether this is thread 0 of the launch's last block, and whether any warp of any block has given up a wait: those blocks count in the upper half, too (no more
// than three blocks an SM: the lower half does not run over).
__device__ __forceinline__ bool last_block(unsigned* done, bool gave_up, bool& broken) {
    broken = __syncthreads_or(gave_up);
    if (threadIdx.x != 0u) return false;
    __threadfence();
    const unsigned before = atomicAdd(done, broken ? 0x10001u : 1u);
    if ((before & 0xFFFFu) + 1u != gridDim.x) return false;
    __threadfence();
    *done = 0u;
    broken = broken || before >> 16;
    return true;
}

// ------------------------------------------------------------------------------------------------ pieces on their way to shared memory
// A piece's arrays as they lie in memory: what is whole blocks of aligned arrays comes by bulk copies, several pieces ahead of the warps that compute; the last,
// shorter block of a tensor, and arrays that are not aligned, those warps load themselves.  Without the copies ahead all warps of the GPU load, then compute, at
// the same time: with moments of 8 bits, whose arithmetic takes as long as their memory traffic, the two times then add up.
struct alignas(16) View {                                                              // a piece of a tensor, addresses at its first value
    const void* grad; const void* weights; void* param; float* master; void* moment1; void* moment2; float* scale1; float* scale2;
    unsigned values, copied, blocks, number;                                 // values of the piece, whole blocks of it that come by copies, blocks, number of the first
    float lr_scale, decay;
    int grad_type, weight_type, param_type;
    bool wide;
};
template <int BITS> struct Stage {
    unsigned char g[WARPS * BLOCK * 4], w[WARPS * BLOCK * 4];
    unsigned char m[WARPS * BLOCK * (BITS / 8)], v[WARPS * BLOCK * (BITS / 8)];
    float scale1[WARPS], scale2[WARPS];
    View view;
};
template <int BITS> struct Ring {
    static constexpr int STAGES = BITS == 32 ? 2 : 3;
    Stage<BITS> stage[STAGES];
    unsigned long long full[STAGES], empty[STAGES];
};
static_assert(sizeof(Stage<8>) % 16 == 0 && sizeof(Stage<32>) % 16 == 0, "bulk copies go to multiples of 16 bytes");
__device__ __forceinline__ void copy4(void* to, const void* from) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" :: "r"(smem_u32(to)), "l"(from) : "memory"); }

template <int BITS> __device__ void init_ring(Ring<BITS>& ring) {
    if (threadIdx.x == 0u)
        for (int i = 0; i < Ring<BITS>::STAGES; ++i) { mbar_init(&ring.full[i], BITS == 8 ? 33u : 1u); mbar_init(&ring.empty[i], WARPS); }
    __syncthreads();
}

// The copying warp (a call of its own: its registers are not the computing warps').  Its lanes look up 32 pieces at a time, then each has its own copied when its turn and a stage come.
// Whoever gives up a wait, this warp returns when what it has begun has landed (or a wait for that has run out, too): until then the block does not end.
template <int BITS> __device__ __noinline__ bool copy_pieces(Ring<BITS>& ring, const Tensor* tensors, const Piece* pieces, unsigned n, Control* ctl) {
    const unsigned lane = threadIdx.x % 32u;
    constexpr unsigned STAGES = Ring<BITS>::STAGES;
    unsigned at = 0u, parity = 1u, begun = 0u;                               // the stage that is next, which phase of `empty` lets it be filled, and pieces so far
    bool fine = true;
    for (unsigned long long base = blockIdx.x; base < n && fine; base += 32ull * gridDim.x) {
        const unsigned long long k = base + (unsigned long long)lane * gridDim.x;
        const Piece pc = k < n ? pieces[k] : Piece{0u, 0u, 0u, 0u};
        const Tensor t = k < n ? tensors[pc.tensor] : Tensor{};
        const long long first = (long long)pc.block * BLOCK;
        const unsigned of_g = t.grad_type == CUDARL_F32 ? 4u : 2u, of_p = t.param_type == CUDARL_F32 ? 4u : 2u, of_w = t.master ? 4u : of_p, of_m = BITS / 8;
        auto moved = [&](void* p, unsigned of) { return p ? static_cast<void*>(static_cast<char*>(p) + first * of) : nullptr; };
        View view;
        view.grad = moved(const_cast<void*>(t.grad), of_g); view.param = moved(t.param, of_p); view.master = static_cast<float*>(moved(t.master, 4u));
        view.weights = t.master ? view.master : view.param;
        view.moment1 = moved(t.moment1, of_m); view.moment2 = moved(t.moment2, of_m);
        view.scale1 = t.scale1 + pc.block; view.scale2 = t.scale2 + pc.block;
        view.values = (unsigned)min(t.count - first, (long long)(WARPS * BLOCK)); view.blocks = pc.blocks; view.number = pc.number;
        view.copied = t.wide && t.copied_grad ? view.values / BLOCK : 0u;
        view.lr_scale = t.lr_scale; view.decay = t.decay;
        view.grad_type = t.grad_type; view.param_type = t.param_type; view.weight_type = t.master ? CUDARL_F32 : t.param_type;
        view.wide = t.wide;
        for (unsigned turn = 0; turn < 32u && base + (unsigned long long)turn * gridDim.x < n && fine; ++turn) {
            Stage<BITS>& st = ring.stage[at];
            unsigned long long* const bar = &ring.full[at];
            // from here on it waits for the computing warps, and they for the norm: how long that takes is not this wait's
            if (begun == STAGES) asm volatile("griddepcontrol.wait;" ::: "memory");
            if (lane == turn) fine = mbar_wait(&ring.empty[at], parity, 0u);
            fine = __shfl_sync(~0u, fine, turn);
            if (!fine) break;
            if (BITS == 8) {                                                 // the scales of its blocks lie anywhere: a lane copies each
                const float* const scale1 = reinterpret_cast<const float*>(__shfl_sync(~0u, reinterpret_cast<unsigned long long>(view.scale1), turn));
                const float* const scale2 = reinterpret_cast<const float*>(__shfl_sync(~0u, reinterpret_cast<unsigned long long>(view.scale2), turn));
                const unsigned blocks = __shfl_sync(~0u, pc.blocks, turn), which = lane % WARPS;
                if (lane < 2u * WARPS && which < blocks) copy4(lane < WARPS ? &st.scale1[which] : &st.scale2[which], (lane < WARPS ? scale1 : scale2) + which);
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(smem_u32(bar)) : "memory");
            }
            if (lane == turn) {
                const unsigned values = view.copied * BLOCK;
                st.view = view;
                mbar_publish_expect_tx(bar, values * (of_g + of_w + 2u * of_m));
                if (values) {
                    bulk_g2s(st.g, view.grad, values * of_g, bar);
                    bulk_g2s(st.w, view.weights, values * of_w, bar);
                    bulk_g2s(st.m, view.moment1, values * of_m, bar);
                    bulk_g2s(st.v, view.moment2, values * of_m, bar);
                }
            }
            __syncwarp();
            ++begun;
            if (++at == STAGES) { at = 0u; parity ^= 1u; }
        }
    }
    for (unsigned i = 0; i < STAGES && i < begun; ++i)                       // the last phase that each stage was begun for
        fine = __all_sync(~0u, mbar_wait(&ring.full[i], ((begun - 1u - i) / STAGES) & 1u, 0u)) && fine;
    if (!fine && lane == 0u) atomicOr(&ctl->error, ERR_COPY_TIMEOUT);
    return fine;
}

// Eight values of a block in a stage: 32 or 16 bytes a lane.
__device__ __forceinline__ void unstage8(Raw& r, const unsigned char* from, int type, unsigned warp, unsigned lane) {
    if (type == CUDARL_F32) {
        const uint4* at = reinterpret_cast<const uint4*>(from) + (warp * 32u + lane) * 2u;
        const uint4 a = at[0], b = at[1];
        r.v[0] = a.x; r.v[1] = a.y; r.v[2] = a.z; r.v[3] = a.w; r.v[4] = b.x; r.v[5] = b.y; r.v[6] = b.z; r.v[7] = b.w;
    } else {
        const uint4 a = reinterpret_cast<const uint4*>(from)[warp * 32u + lane];
        r.v[0] = a.x; r.v[1] = a.y; r.v[2] = a.z; r.v[3] = a.w;
    }
}

// The block's sum in thread 0, always in the same order.
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double warp_sum[WARPS];
    for (int by = 16; by; by /= 2) v += __shfl_xor_sync(~0u, v, by);
    __syncthreads();
    if (threadIdx.x % 32u == 0u) warp_sum[threadIdx.x / 32u] = v;
    __syncthreads();
    v = warp_sum[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) v += warp_sum[w];
    return v;
}
// Squares of eight values of each of COUNT blocks, all loads first.
template <int TYPE, int COUNT> __device__ __forceinline__ void add_squares(double (&sum)[4], const void* grad, long long at) {
    Raw raw[COUNT];
#pragma unroll
    for (int u = 0; u < COUNT; ++u) load8(raw[u], grad, TYPE, at + u * BLOCK, true, 8);
#pragma unroll
    for (int u = 0; u < COUNT; ++u) {
        float g[8];
        floats8(raw[u], TYPE, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i % 4] = fma((double)g[i], (double)g[i], sum[i % 4]);
    }
}

// Sum of squares of all gradients, in 64 bits and in an order that only the list of pieces and the grid make; the last block adds the blocks' sums.  A warp a
// piece, 64 (32 bits) or 128 bytes a lane on their way at a time: as many conversions to 64 bits as take about two thirds of the time that the bytes take.
__global__ void __launch_bounds__(32 * WARPS, 4) k_grad_norm(const Tensor* tensors, const Piece* __restrict__ pieces, unsigned n, Control* ctl, double* part, bool spread, float grad_scale, float max_norm) {
    asm volatile("griddepcontrol.launch_dependents;");                       // the step's blocks may come as these go: they load before they wait for the norm
    double four[4] = {0.0, 0.0, 0.0, 0.0};                                   // (four sums in turn: additions of 64 bits take their time)
    const unsigned lane = threadIdx.x % 32u, warp = threadIdx.x / 32u, stride = gridDim.x * WARPS;
    auto add_block = [&](const Tensor& t, long long at) {                    // one block, or what there is of it
        Raw raw;
        float g[8];
        const int len = (int)min(8ll, t.count - at);
        load8(raw, t.grad, t.grad_type, at, t.wide_grad && len == 8, len);
        floats8(raw, t.grad_type, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) four[i % 4] = fma((double)g[i], (double)g[i], four[i % 4]);
    };
    unsigned k = blockIdx.x * WARPS + warp;                                  // (no overflow: at most 2^26 pieces)
    if (spread) {                                                            // few pieces: a warp a block
        const Piece pc = pieces[blockIdx.x];
        if (warp < pc.blocks) add_block(tensors[pc.tensor], (long long)(pc.block + warp) * BLOCK + lane * 8u);
        k = n;
    }
    Piece next = k < n ? pieces[k] : Piece{0u, 0u, 0u, 0u};
    for (; k < n; k += stride) {
        const Piece pc = next;
        if (k + stride < n) next = pieces[k + stride];
        const Tensor& t = tensors[pc.tensor];
        const int type = t.grad_type;
        const long long first = (long long)pc.block * BLOCK, at = first + lane * 8u;
        if (t.wide_grad && t.count - first >= WARPS * BLOCK) {
            static_assert(WARPS == 8, "the blocks of a whole piece");
            if (type == CUDARL_F32) { add_squares<CUDARL_F32, 4>(four, t.grad, at); add_squares<CUDARL_F32, 4>(four, t.grad, at + 4 * BLOCK); }
            else if (type == CUDARL_BF16) add_squares<CUDARL_BF16, 8>(four, t.grad, at);
            else add_squares<CUDARL_F16, 8>(four, t.grad, at);
        } else
            for (unsigned u = 0; u < pc.blocks; ++u) add_block(t, at + u * BLOCK);
    }
    double sum = block_sum((four[0] + four[1]) + (four[2] + four[3]));
    __shared__ bool last;
    if (threadIdx.x == 0) {
        part[blockIdx.x] = sum;
        __threadfence();
        last = atomicAdd(&ctl->done_norm, 1u) + 1u == gridDim.x;
        __threadfence();
    }
    __syncthreads();
    if (!last) return;
    sum = 0.0;
    for (unsigned b = threadIdx.x; b < gridDim.x; b += 32u * WARPS) sum += __ldcg(part + b);
    sum = block_sum(sum);
    if (threadIdx.x == 0) {
        const double norm = sqrt(sum) * fabs((double)grad_scale);
        ctl->done_norm = 0u;
        ctl->norm = norm;
        ctl->go = isfinite(norm) ? 1u : 0u;
        ctl->clip = (float)fmin(1.0, (double)max_norm / (norm + 1e-6));
    }
}

// |y| <= 448 as an e4m3 code, rounded up or down by 16 random bits: the bits that a code keeps are the float's own above bit 20; below the smallest normal
// code (2^-6) all steps are 2^-9, which adding 2^-6 makes them in the float too.  (Where a warp has only normal codes it makes them four bits higher up, with
// the exponents' difference, 120 << 27 = -0x40000000, in the top byte of the random bits: three instructions a code, and the bytes are picked from the tops.)
__device__ __forceinline__ unsigned to_code(float y, unsigned bits16) {
    const bool small = y < 0.015625f;
    const float z = small ? y + 0.015625f : y;
    return ((__float_as_uint(z) + (bits16 << 4)) >> 20) - (small ? 121u << 3 : 120u << 3);
}
__device__ __forceinline__ float reciprocal_fast(float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float reciprocal_root_fast(float v) { float r; asm("rsqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float max_nan(float a, float b, float c) { float r; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
__device__ __forceinline__ float min3(float a, float b, float c) { float r; asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
__device__ __forceinline__ Two negative2(float v) { return two(-v, -v); }

// Quotients and roots the way of Markstein (1990): an approximation, and its remainder, which a fused multiply-add has exactly, to correct it.
// a / b for |a| <= 448 b; `by` = 1 / b, b in 2^-100 .. 2^100.
__device__ __forceinline__ Two divide2(Two a, float b, float by) {
    const Two by2 = two(by, by), q = mul2(a, by2);
    return fma2(fma2(q, negative2(b), a), by2, q);
}
__device__ __forceinline__ float reciprocal(float b) { const float r = reciprocal_fast(b); return fmaf(r, fmaf(-b, r, 1.0f), r); }
// Zero stays zero (its reciprocal root is infinite, and is made a number).  Below 2^-100 the remainder is not exact any more and the root is what the approximation
// and its product are, 2^-22 of itself off at most; an infinite value gives NaN and is seen to behind this (one test a lane: the reciprocal root is zero there).
__device__ __forceinline__ Two root2(Two v) {
    float a, b;
    apart(v, a, b);
    const Two r = two(fminf(reciprocal_root_fast(a), FLT_MAX), fminf(reciprocal_root_fast(b), FLT_MAX)), q = mul2(v, r), rest = fma2(mul2(q, two(-1.0f, -1.0f)), q, v);
    return fma2(rest, mul2(r, two(0.5f, 0.5f)), q);
}
// What an infinite root is kept as in 8 bits: its square is infinite again, so that the value stays where it is, as with moments of 32 bits -- and its block's scale is a
// number (an infinite one would make NaN of the block's zeros).  Roots of floats end below 2^64.
constexpr float INFINITE_ROOT = 36893488147419103232.0f;                     // 2^65

// A block of threads takes a piece, a warp a block of it, a lane eight values.  Every product and sum of the moments is rounded by itself, and the roots and
// quotients that become codes are correctly rounded (but for one in thousands, off by the last bit, and roots of less than 2^-100): codes do not depend on what a compiler fuses.
template <int BITS>
__global__ void __launch_bounds__(THREADS, RESIDENT) k_adamw(const Tensor* tensors, const Piece* pieces, unsigned n, Control* ctl, const __grid_constant__ Settings s, float lr, float grad_scale) {
    extern __shared__ __align__(128) unsigned char shared_bytes[];
    Ring<BITS>& ring = *reinterpret_cast<Ring<BITS>*>(shared_bytes);
    init_ring(ring);
    const unsigned lane = threadIdx.x % 32u, warp = threadIdx.x / 32u;
    const bool copies = warp == WARPS;
    bool gave_up = false;
    if (s.polls) {                                                           // there are no pieces then: a wait for copies that nobody begins
        gave_up = !__all_sync(~0u, mbar_wait(&ring.full[0], 0u, s.polls));
        if (gave_up && lane == 0u) atomicOr(&ctl->error, ERR_COPY_TIMEOUT);
    }
    if (copies) gave_up = !copy_pieces(ring, tensors, pieces, n, ctl) || gave_up;      // (what it copies is not what the norm's kernel writes)
    asm volatile("griddepcontrol.wait;" ::: "memory");                       // for the norm, when there is one
    const long long step = __ldcg(&ctl->step);
    const float fix1 = __ldcg(&ctl->fix1), root_fix2 = __ldcg(&ctl->root_fix2);
    const bool go = fix1 != 0.0f && (!s.clipped || __ldcg(&ctl->go));        // once a wait has run out, no step does anything
    const float scale = s.clipped ? grad_scale * __ldcg(&ctl->clip) : grad_scale;
    unsigned prefix[4];
    policy_prefix(s.keys, (unsigned long long)(step + 1), prefix);
    unsigned place = 0u, parity = 0u;
    for (unsigned long long k = blockIdx.x; k < n && !copies; k += gridDim.x) {
        Stage<BITS>& st = ring.stage[place];
        unsigned long long* const empty = &ring.empty[place];
        if (!__all_sync(~0u, mbar_wait(&ring.full[place], parity, 0u))) {    // (what is under way the copying warp waits for)
            gave_up = true;
            if (lane == 0u) atomicOr(&ctl->error, ERR_COPY_TIMEOUT);
            break;
        }
        if (++place == Ring<BITS>::STAGES) { place = 0u; parity ^= 1u; }
        const View& view = st.view;
        if (warp < view.blocks && go) {
        const unsigned at = warp * BLOCK + lane * 8u;
        const int len = min(8, (int)view.values - (int)at);                  // of this lane's eight
        const bool wide = view.wide && len == 8;
        const float rate = lr * view.lr_scale, decay = view.decay;
        Raw gr, wr, mr, vr;
        uint2 c1 = make_uint2(0u, 0u), c2 = c1;
        float old1 = 0.0f, old2 = 0.0f;
        if (warp < view.copied) {
            unstage8(gr, st.g, view.grad_type, warp, lane);
            unstage8(wr, st.w, view.weight_type, warp, lane);
            if (BITS == 32) { unstage8(mr, st.m, CUDARL_F32, warp, lane); unstage8(vr, st.v, CUDARL_F32, warp, lane); }
            else { c1 = reinterpret_cast<const uint2*>(st.m)[warp * 32u + lane]; c2 = reinterpret_cast<const uint2*>(st.v)[warp * 32u + lane]; }
        } else {
            load8(gr, view.grad, view.grad_type, at, false, len);
            load8(wr, view.weights, view.weight_type, at, false, len);
            if (BITS == 32) { load8(mr, view.moment1, CUDARL_F32, at, false, len); load8(vr, view.moment2, CUDARL_F32, at, false, len); }
            else { c1 = load_codes(view.moment1, at, false, len); c2 = load_codes(view.moment2, at, false, len); }
        }
        if (BITS == 8) { old1 = st.scale1[warp]; old2 = st.scale2[warp]; }
        float g[8], w[8], m[8], v[8];
        floats8(gr, view.grad_type, g);
        floats8(wr, view.weight_type, w);
        if (BITS == 32) { floats8(mr, CUDARL_F32, m); floats8(vr, CUDARL_F32, v); }
        if (BITS == 8) {
            from_codes(c1.x, m); from_codes(c1.y, m + 4); from_codes(c2.x, v); from_codes(c2.y, v + 4);
            const Two s1 = two(old1, old1), s2 = two(old2, old2);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                apart(mul2(two(m[i], m[i + 1]), s1), m[i], m[i + 1]);
                const Two r = mul2(two(v[i], v[i + 1]), s2);
                apart(mul2(r, r), v[i], v[i + 1]);
            }
        }
        float root[8], top2 = 0.0f;
        const Two one2 = two(s.one, s.one);                                  // (a product by a one that the compiler does not know, plus: a sum that it cannot fuse with the product before)
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const Two gi = mul2(two(g[i], g[i + 1]), two(scale, scale));
            const Two mi = fma2(mul2(two(s.beta1, s.beta1), two(m[i], m[i + 1])), one2, mul2(two(s.rest1, s.rest1), gi));
            const Two vi = fma2(mul2(two(s.beta2, s.beta2), two(v[i], v[i + 1])), one2, mul2(mul2(two(s.rest2, s.rest2), gi), gi));
            apart(mi, m[i], m[i + 1]); apart(vi, v[i], v[i + 1]); apart(root2(vi), root[i], root[i + 1]);
            top2 = max_nan(top2, root[i], root[i + 1]);
        }
        const bool beyond = !(top2 < INFINITE_ROOT);                         // a second moment that is infinite, or NaN
        if (beyond) {
#pragma unroll
            for (int i = 0; i < 8; ++i) root[i] = v[i] == INFINITY ? INFINITY : root[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            float a, b;
            apart(fma2(two(root[i], root[i + 1]), two(root_fix2, root_fix2), two(s.eps, s.eps)), a, b);
            const Two wi = two(w[i], w[i + 1]), way = mul2(mul2(two(m[i], m[i + 1]), two(fix1, fix1)), two(reciprocal_fast(a), reciprocal_fast(b)));
            apart(fma2(negative2(rate), fma2(two(decay, decay), wi, way), wi), w[i], w[i + 1]);
        }
        if (view.master) store8(view.master, CUDARL_F32, at, wide, len, w);
        store8(view.param, view.param_type, at, wide, len, w);
        if (BITS == 32) {
            store8(view.moment1, CUDARL_F32, at, wide, len, m);
            store8(view.moment2, CUDARL_F32, at, wide, len, v);
        } else {
            float top1 = 0.0f;                                               // (values behind the tensor's end are zeros; NaN is the largest)
#pragma unroll
            for (int i = 0; i < 8; i += 2) top1 = max_nan(top1, fabsf(m[i]), fabsf(m[i + 1]));
            if (beyond) {
                top2 = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) { root[i] = root[i] == INFINITY ? INFINITE_ROOT : root[i]; top2 = max_nan(top2, root[i], root[i]); }
            }
            // the largest magnitudes of the block, in the order of their bits
            const float scale1 = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(top1))) * (1.0f / 448.0f), scale2 = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(top2))) * (1.0f / 448.0f);
            if (lane == 0) { view.scale1[warp] = scale1; view.scale2[warp] = scale2; }
            float y1[8], y2[8], least = 448.0f;
            const bool usual = scale1 > 7.9e-31f && scale1 < 1.2e30f && scale2 > 7.9e-31f && scale2 < 1.2e30f;
            if (usual) {
                const float by1 = reciprocal(scale1), by2 = reciprocal(scale2);
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    apart(divide2(two(m[i], m[i + 1]), scale1, by1), y1[i], y1[i + 1]);
                    apart(divide2(two(root[i], root[i + 1]), scale2, by2), y2[i], y2[i + 1]);
                    least = min3(min3(least, fabsf(y1[i]), fabsf(y1[i + 1])), y2[i], y2[i + 1]);
                }
            } else {
                const float by1 = scale1 > 0.0f ? scale1 : 1.0f, by2 = scale2 > 0.0f ? scale2 : 1.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) { y1[i] = m[i] / by1; y2[i] = root[i] / by2; }
            }
            const bool all_normal = __all_sync(~0u, usual && least >= 0.015625f);
            unsigned d1[2], d2[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const U4 r = policy_philox((view.number + warp) * (BLOCK / 4u) + lane * 2u + q, s.keys, prefix);      // counter (quad, 0, step): quads stay below 2^32
                const unsigned word[4] = {r.x, r.y, r.z, r.w};
                unsigned a[4], b[4];                                         // a code in the top byte of each
                if (all_normal) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int e = 4 * q + i;
                        a[i] = (__float_as_uint(y1[e]) << 4) + __byte_perm(word[i], 0x40000000u, 0x7104u) | __float_as_uint(m[e]) & 0x80000000u;
                        b[i] = (__float_as_uint(y2[e]) << 4) + __byte_perm(word[i], 0x40000000u, 0x7324u);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int e = 4 * q + i;
                        a[i] = to_code(fminf(fabsf(y1[e]), 448.0f), word[i] & 0xFFFFu) << 24 | __float_as_uint(m[e]) & 0x80000000u;
                        b[i] = max(to_code(fminf(y2[e], 448.0f), word[i] >> 16), root[e] > 0.0f ? 1u : 0u) << 24;
                    }
                }
                d1[q] = __byte_perm(__byte_perm(a[0], a[1], 0x0073u), __byte_perm(a[2], a[3], 0x0073u), 0x5410u);
                d2[q] = __byte_perm(__byte_perm(b[0], b[1], 0x0073u), __byte_perm(b[2], b[3], 0x0073u), 0x5410u);
            }
            store_codes(view.moment1, at, wide, len, make_uint2(d1[0], d1[1]));
            store_codes(view.moment2, at, wide, len, make_uint2(d2[0], d2[1]));
        }
        }
        __syncwarp();
        if (lane == 0u) mbar_arrive(empty);                                  // the stage can be filled again
    }
    bool broken;
    if (last_block(&ctl->done, gave_up, broken)) {
        if (broken) ctl->fix1 = 0.0f;                                        // a step that was broken off does not count, and is the last
        else if (go) {
            const double p1 = ctl->power1 * s.power1, p2 = ctl->power2 * s.power2;
            ctl->step = step + 1; ctl->power1 = p1; ctl->power2 = p2;
            ctl->fix1 = (float)(1.0 / (1.0 - p1)); ctl->root_fix2 = (float)sqrt(1.0 / (1.0 - p2));
        } else if (fix1 != 0.0f) ctl->skipped += 1;
    }
}

}  // namespace

struct cudarl_adamw {
    cudarl_adamw_config cfg;
    std::vector<Tensor> tensors;
    Tensor* dtensors = nullptr;
    Piece* dpieces = nullptr;
    Control* dctl = nullptr;
    double* dpart = nullptr;
    unsigned pieces = 0, grid = 0, norm_grid = 0;
    bool gradients = false;                  // every tensor with values has one
    unsigned polls = 0;
};

namespace {

size_t ring_bytes(int bits) { return bits == 8 ? sizeof(Ring<8>) : sizeof(Ring<32>); }

int check_tensor(const cudarl_adamw_tensor& t, int bits, CallerArrays& arrays) {
    if (t.count < 0 || t.count > (1ll << 40)) return fail_global(-1, "count of a tensor out of range");
    if (t.param_type < 0 || t.param_type > 2 || t.grad_type < 0 || t.grad_type > 2) return fail_global(-1, "param_type and grad_type must be CUDARL_F32, CUDARL_BF16 or CUDARL_F16");
    if (!(t.lr_scale >= 0.0f) || !std::isfinite(t.lr_scale) || !(t.weight_decay >= 0.0f) || !std::isfinite(t.weight_decay)) return fail_global(-1, "lr_scale and weight_decay must be finite and not negative");
    if (t.count == 0) return 0;
    if (!t.param || !t.moment1 || !t.moment2) return fail_global(-1, "null param or moment");
    if (bits == 8 && (!t.scale1 || !t.scale2)) return fail_global(-1, "moments of 8 bits need their scales");
    int rc;
    const size_t moment = bits == 8 ? 1 : 4;
    if ((rc = arrays.check("param", t.param, type_bytes(t.param_type))) || (rc = arrays.check_if("grad", t.grad, type_bytes(t.grad_type))) || (rc = arrays.check_if("master", t.master, 4)) ||
        (rc = arrays.check("moment1", t.moment1, moment)) || (rc = arrays.check("moment2", t.moment2, moment))) return rc;
    if (bits == 8 && ((rc = arrays.check("scale1", t.scale1, 4)) || (rc = arrays.check("scale2", t.scale2, 4)))) return rc;
    return 0;
}

bool sixteen(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool eight(const void* p, size_t value) { return reinterpret_cast<uintptr_t>(p) % (8 * value) == 0; }

void place_gradient(Tensor& t, const void* grad) {
    t.grad = grad;
    t.copied_grad = sixteen(grad);
    t.wide_grad = eight(grad, type_bytes(t.grad_type));
}

void note_gradients(cudarl_adamw* o) {
    o->gradients = true;
    for (const Tensor& t : o->tensors) o->gradients = o->gradients && (t.grad || t.count == 0);
}

void free_all(cudarl_adamw* o) {
    if (o->dtensors) cudaFree(o->dtensors);
    if (o->dpieces) cudaFree(o->dpieces);
    if (o->dctl) cudaFree(o->dctl);
    if (o->dpart) cudaFree(o->dpart);
}

int fill(cudarl_adamw* o, int32_t count, const cudarl_adamw_tensor* tensors) {
    CurrentDevice current;
    cudaError_t e = current.set(o->cfg.device);
    if (e != cudaSuccess) return fail_cuda("cudaSetDevice", e);
    CallerArrays arrays;
    arrays.expect(o->cfg.device);
    std::vector<Piece> pieces;
    int64_t number = 0;
    for (int32_t i = 0; i < count; ++i) {
        const cudarl_adamw_tensor& t = tensors[i];
        const int rc = check_tensor(t, o->cfg.state_bits, arrays);
        if (rc) return rc;
        Tensor d{t.param, t.grad, t.master, t.moment1, t.moment2, t.scale1, t.scale2, (long long)t.count, t.lr_scale, t.weight_decay, (unsigned char)t.param_type, (unsigned char)t.grad_type, 0, 0, 0};
        const size_t moment = o->cfg.state_bits == 8 ? 1 : 4;
        d.wide = eight(t.param, type_bytes(t.param_type)) && eight(t.master, 4) && sixteen(t.moment1) && sixteen(t.moment2) && eight(t.moment1, moment) && eight(t.moment2, moment);
        place_gradient(d, t.grad);
        o->tensors.push_back(d);
        const int64_t blocks = (t.count + BLOCK - 1) / BLOCK;
        if (number + blocks > (1ll << 26)) return fail_global(-1, "more than 2^34 values in one handle");
        for (int64_t b = 0; b < blocks; b += WARPS) pieces.push_back(Piece{(unsigned)i, (unsigned)b, (unsigned)std::min<int64_t>(WARPS, blocks - b), (unsigned)(number + b)});
        number += blocks;
    }
    note_gradients(o);
    o->pieces = (unsigned)pieces.size();
    const int bits = o->cfg.state_bits;
    if ((e = bits == 32 ? cudaFuncSetAttribute(k_adamw<32>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ring_bytes(32))
                        : cudaFuncSetAttribute(k_adamw<8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ring_bytes(8))) != cudaSuccess) return fail_cuda("cudaFuncSetAttribute", e);
    int sms = 0;
    if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, o->cfg.device)) != cudaSuccess) return fail_cuda("cudaDeviceGetAttribute", e);
    const unsigned most = (unsigned)(sms * RESIDENT), blocks = o->pieces;
    o->grid = blocks < 1u ? 1u : blocks < most ? blocks : most;
    const unsigned norm_most = (unsigned)(sms * 4);                          // a block of threads a piece where there are so few, else a warp
    o->norm_grid = o->pieces < 1u ? 1u : o->pieces < norm_most ? o->pieces : norm_most;
    Control c;
    std::memset(&c, 0, sizeof c);
    c.step = o->cfg.step;
    c.power1 = std::pow(o->cfg.beta1, (double)(c.step + 1));
    c.power2 = std::pow(o->cfg.beta2, (double)(c.step + 1));
    c.fix1 = (float)(1.0 / (1.0 - c.power1)); c.root_fix2 = (float)std::sqrt(1.0 / (1.0 - c.power2));
    c.clip = 1.0f;
    if ((e = cudaMalloc(&o->dtensors, sizeof(Tensor) * (o->tensors.size() + 1))) != cudaSuccess || (e = cudaMalloc(&o->dpieces, sizeof(Piece) * (pieces.size() + 1))) != cudaSuccess ||
        (e = cudaMalloc(&o->dctl, sizeof(Control))) != cudaSuccess || (e = cudaMalloc(&o->dpart, sizeof(double) * o->norm_grid)) != cudaSuccess) return fail_cuda("cudaMalloc", e);
    if ((e = cudaMemcpy(o->dtensors, o->tensors.data(), sizeof(Tensor) * o->tensors.size(), cudaMemcpyHostToDevice)) != cudaSuccess ||
        (e = cudaMemcpy(o->dpieces, pieces.data(), sizeof(Piece) * pieces.size(), cudaMemcpyHostToDevice)) != cudaSuccess ||
        (e = cudaMemcpy(o->dctl, &c, sizeof c, cudaMemcpyHostToDevice)) != cudaSuccess || (e = cudaDeviceSynchronize()) != cudaSuccess) return fail_cuda("cudaMemcpy", e);
    return 0;
}

}  // namespace

extern "C" int cudarl_adamw_create(const cudarl_adamw_config* cfg, int32_t count, const cudarl_adamw_tensor* tensors, cudarl_adamw** out) {
    if (!cfg || !out || (count > 0 && !tensors)) return fail_global(-1, "null argument");
    *out = nullptr;
    if (cfg->struct_size != sizeof(cudarl_adamw_config)) return fail_global(-1, "cudarl_adamw_config.struct_size mismatch");
    if (count < 0) return fail_global(-1, "count negative");
    if (cfg->device < 0) return fail_global(-1, "device negative");
    if (cfg->state_bits != 32 && cfg->state_bits != 8) return fail_global(-1, "state_bits must be 32 or 8");
    if (!(cfg->beta1 >= 0.0 && cfg->beta1 < 1.0) || !(cfg->beta2 >= 0.0 && cfg->beta2 < 1.0)) return fail_global(-1, "beta1 and beta2 must be in [0, 1)");
    if (!(cfg->eps >= 1e-30) || !(cfg->eps <= 1e30)) return fail_global(-1, "eps must be in 1e-30 .. 1e30");
    if (!(cfg->max_grad_norm >= 0.0f) || !std::isfinite(cfg->max_grad_norm)) return fail_global(-1, "max_grad_norm must be finite and not negative");
    if (cfg->step < 0 || cfg->step > (1ll << 62)) return fail_global(-1, "step out of range");
    cudarl_adamw* o = new (std::nothrow) cudarl_adamw();
    if (!o) return fail_global(-1, "out of host memory");
    o->cfg = *cfg;
    int rc;
    try { rc = fill(o, count, tensors); } catch (const std::bad_alloc&) { rc = fail_global(-1, "out of host memory"); } catch (...) { rc = fail_global(-1, "unexpected exception"); }
    if (rc) { free_all(o); delete o; return rc; }
    *out = o;
    return 0;
}

extern "C" void cudarl_adamw_destroy(cudarl_adamw* o) {
    if (!o) return;
    CurrentDevice current;
    if (current.set(o->cfg.device) == cudaSuccess) { cudaDeviceSynchronize(); free_all(o); }
    delete o;
}

extern "C" int cudarl_adamw_step(cudarl_adamw* o, float lr, float grad_scale, void* stream) {
    if (!o) return fail_global(-1, "null argument");
    if (!(lr >= 0.0f) || !std::isfinite(lr)) return fail_global(-1, "lr must be finite and not negative");
    if (!std::isfinite(grad_scale)) return fail_global(-1, "grad_scale must be finite");
    if (!o->gradients) return fail_global(-1, "a tensor has no gradient");
    CurrentDevice current;
    cudaError_t e = current.set(o->cfg.device);
    if (e != cudaSuccess) return fail_cuda("cudaSetDevice", e);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudarl_adamw_config& c = o->cfg;
    Settings s{(float)c.beta1, (float)(1.0 - c.beta1), (float)c.beta2, (float)(1.0 - c.beta2), (float)c.eps, 1.0f, {}, c.max_grad_norm > 0.0f, o->polls, c.beta1, c.beta2};
    for (unsigned r = 0; r < 10; ++r) {
        s.keys[2 * r] = (unsigned)c.seed + r * 0x9E3779B9u;
        s.keys[2 * r + 1] = ((unsigned)(c.seed >> 32) ^ TAG_OPTIMIZER) + r * 0xBB67AE85u;
    }
    if (s.clipped) {
        if ((e = launch(k_grad_norm, o->norm_grid, 32 * WARPS, st, o->dtensors, o->dpieces, o->pieces, o->dctl, o->dpart, o->norm_grid == o->pieces, grad_scale, c.max_grad_norm)) != cudaSuccess)
            return fail_cuda("cudarl_adamw_step", e);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(o->grid); cfg.blockDim = dim3(THREADS); cfg.stream = st;
    cfg.dynamicSmemBytes = ring_bytes(c.state_bits);
    // after the norm's kernel: started while that one still runs, its first loads done, it waits for the norm on the device.  Without a norm it must not begin
    // before the gradients' own kernel has ended
    cudaLaunchAttribute early[1];
    early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization; early[0].val.programmaticStreamSerializationAllowed = 1;
    if (s.clipped) { cfg.attrs = early; cfg.numAttrs = 1; }
    const Tensor* tensors = o->dtensors;
    const Piece* pieces = o->dpieces;
    const unsigned n = o->polls ? 0u : o->pieces;
    e = c.state_bits == 32 ? cudaLaunchKernelEx(&cfg, k_adamw<32>, tensors, pieces, n, o->dctl, s, lr, grad_scale)
                           : cudaLaunchKernelEx(&cfg, k_adamw<8>, tensors, pieces, n, o->dctl, s, lr, grad_scale);
    return e == cudaSuccess ? 0 : fail_cuda("cudarl_adamw_step", e);
}

extern "C" int cudarl_adamw_set_gradients(cudarl_adamw* o, const void* const* grads, void* stream) {
    if (!o || (!grads && !o->tensors.empty())) return fail_global(-1, "null argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    CurrentDevice current;
    cudaError_t e = current.set(o->cfg.device);
    if (e != cudaSuccess) return fail_cuda("cudaSetDevice", e);
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if ((e = cudaStreamIsCapturing(st, &capture)) != cudaSuccess) return fail_cuda("cudaStreamIsCapturing", e);
    if (capture != cudaStreamCaptureStatusNone) return fail_global(-1, "gradients cannot be set while the stream is captured");
    CallerArrays arrays;
    arrays.expect(o->cfg.device);
    for (size_t i = 0; i < o->tensors.size(); ++i) {
        if (o->tensors[i].count == 0) continue;
        if (!grads[i]) return fail_global(-1, "null gradient");
        const int rc = arrays.check("grad", grads[i], type_bytes(o->tensors[i].grad_type));
        if (rc) return rc;
    }
    for (size_t i = 0; i < o->tensors.size(); ++i) {
        Tensor& t = o->tensors[i];
        place_gradient(t, grads[i]);
    }
    note_gradients(o);
    // the copy is from pageable memory: it has been taken from there when the call returns
    if (!o->tensors.empty() && (e = cudaMemcpyAsync(o->dtensors, o->tensors.data(), sizeof(Tensor) * o->tensors.size(), cudaMemcpyHostToDevice, st)) != cudaSuccess) return fail_cuda("cudaMemcpyAsync", e);
    return 0;
}

extern "C" int cudarl_adamw_get_stats(cudarl_adamw* o, cudarl_adamw_stats* out) {
    if (!o || !out) return fail_global(-1, "null argument");
    CurrentDevice current;
    cudaError_t e = current.set(o->cfg.device);
    if (e != cudaSuccess) return fail_cuda("cudaSetDevice", e);
    Control c;
    if ((e = cudaDeviceSynchronize()) != cudaSuccess || (e = cudaMemcpy(&c, o->dctl, sizeof c, cudaMemcpyDeviceToHost)) != cudaSuccess) return fail_cuda("cudarl_adamw_get_stats", e);
    out->step = c.step; out->skipped = c.skipped; out->grad_norm = c.norm;
    if (c.error) return fail_global(CUDARL_ERR_DEVICE + (int)c.error, "a wait of the optimizer's kernel ran out: its tensors are not to be used");
    return 0;
}

extern "C" int cudarl_debug_adamw_set_copy_wait_polls(cudarl_adamw* o, int32_t polls) {
    if (!o) return fail_global(-1, "null argument");
    if (polls < 0) return fail_global(-1, "polls negative");
    o->polls = (unsigned)polls;
    return 0;
}
