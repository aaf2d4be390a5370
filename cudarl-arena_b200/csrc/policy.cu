// policy.cu -- log probabilities of the actions taken, entropy and most probable alternatives of rows of logits, and the gradient of the logits.
//
// Row x, legal actions L, c = 1 / temperature, m = max x:   d = (x - m) c <= 0,   S = sum e^d,   log p = d - log S,
//   H = log S - (sum d e^d) / S        (both terms >= 0: nothing cancels)
//   dx_j = c (gl ([j = taken] - p_j) - gH p_j (log p_j + H))
// The statistics of a row for its gradient: {m, log S, H}.
#include "caller_arrays.cuh"

namespace {
using namespace cudarl;

constexpr float NONE = -INFINITY;

struct Rows {
    const void* logits;
    const unsigned char* legal;
    const int* taken;
    long long rows, stride, legal_stride;
    int actions;
    float scale;                       // 1 / temperature
};

constexpr int THREADS = 256;

template <class F> __device__ float block_fold(float v, F f) {
    __shared__ float part[THREADS / 32];
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(~0u, v, o));
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < THREADS / 32; ++i) v = f(v, part[i]);
    return v;
}
__device__ unsigned long long block_max64(unsigned long long v) {
    __shared__ unsigned long long part[THREADS / 32];
    for (int o = 16; o; o >>= 1) v = max(v, __shfl_xor_sync(~0u, v, o));
    __syncthreads();
    if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < THREADS / 32; ++i) v = max(v, part[i]);
    return v;
}

// Larger for the larger logit, of equal ones for the lower action; 0 for none.
__device__ __forceinline__ unsigned long long order_key(float x, unsigned action) {
    const unsigned b = __float_as_uint(x + 0.0f);                            // -0 counts as 0
    return ((unsigned long long)((b & 0x80000000u) ? ~b : b | 0x80000000u) << 32) | (0xFFFFFFFFu - action);
}

template <int TYPE>
__global__ void __launch_bounds__(THREADS) k_logprobs(Rows p, float* logprob, float* entropy, float4* stats, int top, int* top_actions, float* top_logprobs) {
    using O = Of<TYPE>;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const auto* x = static_cast<const typename O::T*>(p.logits) + r * p.stride;
        const unsigned char* legal = p.legal ? p.legal + r * p.legal_stride : nullptr;
        auto at = [&](int j) { return legal && !legal[j] ? NONE : O::get(x[j]); };
        float m = NONE;
        for (int j = threadIdx.x; j < p.actions; j += THREADS) m = fmaxf(m, at(j));
        m = block_fold(m, [](float a, float b) { return fmaxf(a, b); });
        const float from = m == NONE ? 0.0f : m;
        float s = 0.0f, t = 0.0f;
        for (int j = threadIdx.x; j < p.actions; j += THREADS) {
            const float d = (at(j) - from) * p.scale, e = __expf(d);
            s += e;
            if (e > 0.0f) t += d * e;
        }
        s = block_fold(s, [](float a, float b) { return a + b; });
        t = block_fold(t, [](float a, float b) { return a + b; });
        const bool nothing = s == 0.0f, bad = !(s == s);
        const float log_s = logf(s), h = nothing ? 0.0f : log_s - t / s;
        if (threadIdx.x == 0) {
            if (logprob) {
                const int a = p.taken ? p.taken[r] : -1;
                logprob[r] = bad ? s : (unsigned)a >= (unsigned)p.actions ? 0.0f : nothing ? NONE : (at(a) - m) * p.scale - log_s;
            }
            if (entropy) entropy[r] = h;
            if (stats) stats[r] = make_float4(m, log_s, h, 0.0f);
        }
        unsigned long long below = ~0ull;
        for (int k = 0; k < top; ++k) {
            unsigned long long best = 0ull;
            if (!nothing && !bad)
                for (int j = threadIdx.x; j < p.actions; j += THREADS) {
                    const float v = at(j);
                    const unsigned long long key = order_key(v, (unsigned)j);
                    if (v > NONE && key < below && key > best) best = key;
                }
            best = block_max64(best);
            if (threadIdx.x == 0) {
                const int a = best ? (int)(0xFFFFFFFFu - (unsigned)best) : -1;
                top_actions[r * top + k] = a;
                top_logprobs[r * top + k] = bad ? s : best ? (at(a) - m) * p.scale - log_s : NONE;
            }
            below = best;
        }
    }
}

template <int TYPE>
__global__ void __launch_bounds__(THREADS) k_logprobs_backward(Rows p, const float4* stats, const float* grad_logprob, const float* grad_entropy, void* grad, long long grad_stride) {
    using O = Of<TYPE>;
    for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const auto* x = static_cast<const typename O::T*>(p.logits) + r * p.stride;
        auto* g = static_cast<typename O::T*>(grad) + r * grad_stride;
        const unsigned char* legal = p.legal ? p.legal + r * p.legal_stride : nullptr;
        const float4 st = stats[r];
        const int a = p.taken ? p.taken[r] : -1;
        const float gl = (unsigned)a < (unsigned)p.actions && grad_logprob ? grad_logprob[r] : 0.0f, gh = grad_entropy ? grad_entropy[r] : 0.0f;
        for (int j = threadIdx.x; j < p.actions; j += THREADS) {
            float v = 0.0f;
            if ((!legal || legal[j]) && st.y != NONE) {
                const float lp = fmaxf((O::get(x[j]) - st.x) * p.scale - st.y, -1e30f), pr = __expf(lp);
                v = p.scale * (gl * (j == a ? -expm1f(lp) : -pr) - gh * pr * (lp + st.z));
                if (!(st.y == st.y)) v = st.y;
            }
            g[j] = O::put(v);
        }
    }
}

int check_rows(const cudarl_policy_rows* p) {
    if (!p) return fail_global(-1, "null argument");
    if (p->struct_size != sizeof(cudarl_policy_rows)) return fail_global(-1, "cudarl_policy_rows.struct_size mismatch");
    if (p->type != CUDARL_F32 && p->type != CUDARL_BF16 && p->type != CUDARL_F16) return fail_global(-1, "type must be CUDARL_F32, CUDARL_BF16 or CUDARL_F16");
    if (p->rows < 0 || p->actions < 1 || p->actions > 0x7FFFFFFFll) return fail_global(-1, "rows or actions out of range");
    if (p->row_stride < p->actions) return fail_global(-1, "row_stride smaller than a row");
    if (p->legal && p->legal_stride != 0 && p->legal_stride < p->actions) return fail_global(-1, "legal_stride must be 0 or at least a row");
    const int64_t widest = p->row_stride > p->legal_stride ? p->row_stride : p->legal_stride;
    if (p->rows > (1ll << 40) || widest > (1ll << 40) || p->rows > (1ll << 56) / widest) return fail_global(-1, "rows or strides out of range");
    if (!(p->inv_temperature > 0.0f) || p->inv_temperature > 3.4e38f) return fail_global(-1, "inv_temperature must be positive and finite");
    if (p->rows > 0 && !p->logits) return fail_global(-1, "null logits");
    return 0;
}

Rows device_rows(const cudarl_policy_rows* p) {
    return Rows{p->logits, p->legal, p->taken, (long long)p->rows, (long long)p->row_stride, (long long)p->legal_stride, (int)p->actions, p->inv_temperature};
}

unsigned grid_of(long long rows) { return (unsigned)(rows < (1ll << 30) ? rows : (1ll << 30)); }

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
    cudaError_t e = current.set(arrays.device());
    if (e != cudaSuccess) return fail_cuda("cudaSetDevice", e);
    const Rows r = device_rows(p);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned grid = grid_of(r.rows);
    float4* s4 = reinterpret_cast<float4*>(stats);
    switch (p->type) {
    case CUDARL_F32: k_logprobs<CUDARL_F32><<<grid, THREADS, 0, st>>>(r, logprob, entropy, s4, top, top_actions, top_logprobs); break;
    case CUDARL_BF16: k_logprobs<CUDARL_BF16><<<grid, THREADS, 0, st>>>(r, logprob, entropy, s4, top, top_actions, top_logprobs); break;
    default: k_logprobs<CUDARL_F16><<<grid, THREADS, 0, st>>>(r, logprob, entropy, s4, top, top_actions, top_logprobs); break;
    }
    e = cudaGetLastError();
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
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned grid = grid_of(r.rows);
    const float4* s4 = reinterpret_cast<const float4*>(stats);
    switch (p->type) {
    case CUDARL_F32: k_logprobs_backward<CUDARL_F32><<<grid, THREADS, 0, st>>>(r, s4, grad_logprob, grad_entropy, grad_logits, grad_stride); break;
    case CUDARL_BF16: k_logprobs_backward<CUDARL_BF16><<<grid, THREADS, 0, st>>>(r, s4, grad_logprob, grad_entropy, grad_logits, grad_stride); break;
    default: k_logprobs_backward<CUDARL_F16><<<grid, THREADS, 0, st>>>(r, s4, grad_logprob, grad_entropy, grad_logits, grad_stride); break;
    }
    e = cudaGetLastError();
    return e == cudaSuccess ? 0 : fail_cuda("cudarl_policy_logprobs_backward", e);
}
