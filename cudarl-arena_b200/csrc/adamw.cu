// adamw.cu -- one AdamW step over all tensors of a network, moments in 32 bits or in 8, with clipping by the global norm.
//
// The handle keeps on the device: the list of the tensors, a list of the pieces of them that one warp takes at a time (256 values, the block of one
// scale of the 8-bit moments), and the step count with what depends on it.  Nothing of a step comes from the host but lr and grad_scale, so a
// captured step counts on.
#include "caller_arrays.cuh"
#include "rules.cuh"
#include <cuda_fp8.h>
#include <cmath>
#include <cstring>
#include <new>
#include <vector>

namespace {
using namespace cudarl;

constexpr unsigned TAG_OPTIMIZER = 0x4F50544Du;
constexpr int BLOCK = CUDARL_ADAMW_BLOCK;
constexpr int WARPS = 8, THREADS = 32 * WARPS;

struct Tensor {
    void* param; const void* grad; float* master; void* moment1; void* moment2; float* scale1; float* scale2;
    long long count;
    int param_type, grad_type;
    float lr_scale, decay;
};
struct Piece { unsigned tensor, block; };     // the tensor's values block * 256 ...

struct Control {
    long long step, skipped;
    double norm, power1, power2;              // powers of the betas for the step to come
    float clip;
    unsigned go;                              // 0: the norm was no finite number
    unsigned done, done_norm;                 // blocks of the launch that have finished
};

struct Settings { float beta1, rest1, beta2, rest2, eps; unsigned k0, k1; int clipped; double power1, power2; };   // rest = 1 - beta

__device__ __forceinline__ float load(const void* p, int type, long long i) {
    if (type == CUDARL_F32) return static_cast<const float*>(p)[i];
    if (type == CUDARL_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store(void* p, int type, long long i, float v) {
    if (type == CUDARL_F32) static_cast<float*>(p)[i] = v;
    else if (type == CUDARL_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(p)[i] = __float2half_rn(v);
}

__device__ __forceinline__ bool last_block(unsigned* done) {
    __syncthreads();
    if (threadIdx.x != 0u) return false;
    __threadfence();
    if (atomicAdd(done, 1u) + 1u != gridDim.x) return false;
    __threadfence();
    *done = 0u;
    return true;
}

// Sum of squares of all gradients, in 64 bits and in an order that only the list of pieces and the grid make; the last block adds the blocks' sums.
__global__ void __launch_bounds__(THREADS) k_grad_norm(const Tensor* tensors, const Piece* pieces, unsigned n, Control* ctl, double* part, float grad_scale, float max_norm) {
    double sum = 0.0;
    const unsigned lane = threadIdx.x % 32u, warp = threadIdx.x / 32u;
    for (unsigned k = blockIdx.x * WARPS + warp; k < n; k += gridDim.x * WARPS) {
        const Piece pc = pieces[k];
        const Tensor& t = tensors[pc.tensor];
        const long long from = (long long)pc.block * BLOCK;
        const int len = (int)min((long long)BLOCK, t.count - from);
        for (int i = lane; i < len; i += 32) { const double g = load(t.grad, t.grad_type, from + i); sum += g * g; }
    }
    __shared__ double shared[THREADS];
    shared[threadIdx.x] = sum;
    __syncthreads();
    for (unsigned o = THREADS / 2; o; o >>= 1) {
        if (threadIdx.x < o) shared[threadIdx.x] += shared[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) part[blockIdx.x] = shared[0];
    __shared__ bool last;
    const bool l = last_block(&ctl->done_norm);
    if (threadIdx.x == 0) last = l;
    __syncthreads();
    if (!last) return;
    sum = 0.0;
    for (unsigned b = threadIdx.x; b < gridDim.x; b += THREADS) sum += __ldcg(part + b);
    shared[threadIdx.x] = sum;
    __syncthreads();
    for (unsigned o = THREADS / 2; o; o >>= 1) {
        if (threadIdx.x < o) shared[threadIdx.x] += shared[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const double norm = sqrt(shared[0]) * fabs((double)grad_scale);
        ctl->norm = norm;
        ctl->go = isfinite(norm) ? 1u : 0u;
        ctl->clip = (float)fmin(1.0, (double)max_norm / (norm + 1e-6));
    }
}

__device__ __forceinline__ float warp_max(float v) {
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
    return v;
}

// |y| <= 448 as an e4m3 code, rounded up or down by 16 random bits: the bits that a code keeps are the float's own above bit 20; below the smallest normal
// code (2^-6) all steps are 2^-9, which adding 2^-6 makes them in the float too.
__device__ __forceinline__ unsigned to_code(float y, unsigned bits16) {
    const bool small = y < 0.015625f;
    const float z = small ? y + 0.015625f : y;
    return ((__float_as_uint(z) + (bits16 << 4)) >> 20) - (small ? 121u << 3 : 120u << 3);
}
__device__ __forceinline__ float from_code(unsigned char c) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
}

template <int BITS>
__global__ void __launch_bounds__(THREADS) k_adamw(const Tensor* tensors, const Piece* pieces, unsigned n, Control* ctl, Settings s, float lr, float grad_scale) {
    const unsigned lane = threadIdx.x % 32u, warp = threadIdx.x / 32u;
    const long long step = ctl->step;
    const bool go = !s.clipped || ctl->go;
    const float fix1 = (float)(1.0 / (1.0 - ctl->power1)), fix2 = (float)(1.0 / (1.0 - ctl->power2));
    const float scale = s.clipped ? grad_scale * ctl->clip : grad_scale;
    for (unsigned k = blockIdx.x * WARPS + warp; go && k < n; k += gridDim.x * WARPS) {
        const Piece pc = pieces[k];
        const Tensor& t = tensors[pc.tensor];
        const long long from = (long long)pc.block * BLOCK;
        const int len = (int)min((long long)BLOCK, t.count - from);
        float m[8], v[8], scale1 = 0.0f, scale2 = 0.0f;
        if (BITS == 8) { scale1 = t.scale1[pc.block]; scale2 = t.scale2[pc.block]; }
        float top1 = 0.0f, top2 = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int j = (int)lane + 32 * i;
            m[i] = v[i] = 0.0f;
            if (j >= len) continue;
            const long long at = from + j;
            const float g = load(t.grad, t.grad_type, at) * scale;
            float w = t.master ? t.master[at] : load(t.param, t.param_type, at);
            if (BITS == 32) { m[i] = static_cast<float*>(t.moment1)[at]; v[i] = static_cast<float*>(t.moment2)[at]; }
            else {
                m[i] = from_code(static_cast<unsigned char*>(t.moment1)[at]) * scale1;
                const float root = from_code(static_cast<unsigned char*>(t.moment2)[at]) * scale2;
                v[i] = root * root;
            }
            m[i] = s.beta1 * m[i] + s.rest1 * g;
            v[i] = s.beta2 * v[i] + s.rest2 * g * g;
            w -= lr * t.lr_scale * (t.decay * w + m[i] * fix1 / (sqrtf(v[i] * fix2) + s.eps));
            if (t.master) t.master[at] = w;
            store(t.param, t.param_type, at, w);
            if (BITS == 32) { static_cast<float*>(t.moment1)[at] = m[i]; static_cast<float*>(t.moment2)[at] = v[i]; }
            else { v[i] = sqrtf(v[i]); top1 = fmaxf(top1, fabsf(m[i])); top2 = fmaxf(top2, v[i]); }
        }
        if (BITS == 8) {
            scale1 = warp_max(top1) / 448.0f; scale2 = warp_max(top2) / 448.0f;
            if (lane == 0) { t.scale1[pc.block] = scale1; t.scale2[pc.block] = scale2; }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int j = (int)lane + 32 * i;
                if (j >= len) continue;
                const unsigned long long quad = (unsigned long long)k * (BLOCK / 4) + (unsigned)j / 4u;
                const U4 r = philox4x32_10((unsigned)quad, (unsigned)(quad >> 32), (unsigned)(step + 1), (unsigned)((unsigned long long)(step + 1) >> 32), s.k0, s.k1);
                const unsigned word = j % 4 == 0 ? r.x : j % 4 == 1 ? r.y : j % 4 == 2 ? r.z : r.w;
                const unsigned c1 = to_code(fminf(fabsf(m[i]) / (scale1 > 0.0f ? scale1 : 1.0f), 448.0f), word & 0xFFFFu);
                unsigned c2 = to_code(fminf(v[i] / (scale2 > 0.0f ? scale2 : 1.0f), 448.0f), word >> 16);
                if (c2 == 0u && v[i] > 0.0f) c2 = 1u;
                static_cast<unsigned char*>(t.moment1)[from + j] = (unsigned char)(c1 | (m[i] < 0.0f ? 128u : 0u));
                static_cast<unsigned char*>(t.moment2)[from + j] = (unsigned char)c2;
            }
        }
    }
    if (last_block(&ctl->done)) {
        if (go) { ctl->step = step + 1; ctl->power1 *= s.power1; ctl->power2 *= s.power2; }
        else ctl->skipped += 1;
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
    unsigned pieces = 0, grid = 0;
    bool gradients = false;                  // every tensor with values has one
};

namespace {

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
    for (int32_t i = 0; i < count; ++i) {
        const cudarl_adamw_tensor& t = tensors[i];
        const int rc = check_tensor(t, o->cfg.state_bits, arrays);
        if (rc) return rc;
        o->tensors.push_back(Tensor{t.param, t.grad, t.master, t.moment1, t.moment2, t.scale1, t.scale2, (long long)t.count, t.param_type, t.grad_type, t.lr_scale, t.weight_decay});
        const int64_t blocks = (t.count + BLOCK - 1) / BLOCK;
        if ((int64_t)pieces.size() + blocks > (1ll << 31)) return fail_global(-1, "more than 2^39 values in one handle");
        for (int64_t b = 0; b < blocks; ++b) pieces.push_back(Piece{(unsigned)i, (unsigned)b});
    }
    note_gradients(o);
    o->pieces = (unsigned)pieces.size();
    int sms = 0;
    if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, o->cfg.device)) != cudaSuccess) return fail_cuda("cudaDeviceGetAttribute", e);
    const unsigned most = (unsigned)sms * 8u, blocks = (o->pieces + WARPS - 1) / WARPS;
    o->grid = blocks < 1u ? 1u : blocks < most ? blocks : most;
    Control c;
    std::memset(&c, 0, sizeof c);
    c.step = o->cfg.step;
    c.power1 = std::pow(o->cfg.beta1, (double)(c.step + 1));
    c.power2 = std::pow(o->cfg.beta2, (double)(c.step + 1));
    c.clip = 1.0f;
    if ((e = cudaMalloc(&o->dtensors, sizeof(Tensor) * (o->tensors.size() + 1))) != cudaSuccess || (e = cudaMalloc(&o->dpieces, sizeof(Piece) * (pieces.size() + 1))) != cudaSuccess ||
        (e = cudaMalloc(&o->dctl, sizeof(Control))) != cudaSuccess || (e = cudaMalloc(&o->dpart, sizeof(double) * o->grid)) != cudaSuccess) return fail_cuda("cudaMalloc", e);
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
    const Settings s{(float)c.beta1, (float)(1.0 - c.beta1), (float)c.beta2, (float)(1.0 - c.beta2), (float)c.eps, (unsigned)c.seed, (unsigned)(c.seed >> 32) ^ TAG_OPTIMIZER,
                     c.max_grad_norm > 0.0f, c.beta1, c.beta2};
    if (s.clipped) k_grad_norm<<<o->grid, THREADS, 0, st>>>(o->dtensors, o->dpieces, o->pieces, o->dctl, o->dpart, grad_scale, c.max_grad_norm);
    if (c.state_bits == 32) k_adamw<32><<<o->grid, THREADS, 0, st>>>(o->dtensors, o->dpieces, o->pieces, o->dctl, s, lr, grad_scale);
    else k_adamw<8><<<o->grid, THREADS, 0, st>>>(o->dtensors, o->dpieces, o->pieces, o->dctl, s, lr, grad_scale);
    e = cudaGetLastError();
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
    for (size_t i = 0; i < o->tensors.size(); ++i) o->tensors[i].grad = grads[i];
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
    return 0;
}
