// Row-wise kernels of the 8-bit path: the quantiser of activations, and the norm block (norms behind and in front of a block with its gate and
// residual scales, the result in 16 or 32 bits or as 8-bit codes).
#include "elem.cuh"
#include "ptx_utils.cuh"
#include "q8.cuh"

namespace b200 {
namespace {

constexpr int kRowThreads = 256;

// Reductions over a block; `s_part` has a word per warp and is free again behind the next barrier.
template <typename T, typename F>
__device__ __forceinline__ T block_reduce(T v, T* s_part, F&& f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s_part[0];
#pragma unroll
    for (int i = 1; i < kRowThreads / 32; ++i) v = f(v, s_part[i]);
    return v;
}
__device__ __forceinline__ float block_sum(float v, float* s_part) { return block_reduce(v, s_part, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* s_part) { return block_reduce(v, s_part, [](uint32_t a, uint32_t b) { return max(a, b); }); }

// A block per row, two passes over it.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
q8_quantize_kernel(const T* __restrict__ x, long long ldx, int cols, int8_t* __restrict__ codes, long long ldc, int pad_to, float* __restrict__ scales) {
    __shared__ uint32_t s_max[kRowThreads / 32];
    pdl_enter();
    const T* row = x + blockIdx.x * ldx;
    int8_t* out = codes + blockIdx.x * ldc;
    uint32_t m = 0;
    for (int c = threadIdx.x; c < cols; c += kRowThreads) m = max(m, q8_abs_bits(to_f32(row[c])));
    const Q8Row q = q8_row(block_max(m, s_max));
    for (int c = threadIdx.x; c < cols; c += kRowThreads) out[c] = (int8_t)q8_code(to_f32(row[c]), q.inv);
    for (int c = cols + threadIdx.x; c < pad_to; c += kRowThreads) out[c] = 0;
    if (threadIdx.x == 0) scales[blockIdx.x] = q.scale;
}

__device__ __forceinline__ float gate_value(float g, int kind) { return kind == B200ATTN_GATE_SIGMOID ? 1.0f / (1.0f + expf(-g)) : g; }

// A block per row, the updated row in shared memory between the passes.  Products and sums of the update are rounded one by one: the codes then are
// what the formula gives in 32 bits, whatever contracts there.
template <typename X, typename T>
__global__ void __launch_bounds__(kRowThreads)
norm_block_kernel(const b200attn_norm_args a) {
    extern __shared__ float s_row[];
    __shared__ float s_sum[2][kRowThreads / 32];
    __shared__ uint32_t s_max[kRowThreads / 32];
    pdl_enter();
    const long long row = blockIdx.x;
    const X* x = static_cast<const X*>(a.d_x) + row * a.ldx;
    const T* y = static_cast<const T*>(a.d_y) + row * a.ldy;
    const T* g = static_cast<const T*>(a.d_gate) + row * a.ld_gate;
    X* x_out = static_cast<X*>(a.d_x_out) + row * a.ldx_out;
    float post = 1.f;
    if (a.d_post_w) {
        float ss = 0.f;
        for (int c = threadIdx.x; c < a.width; c += kRowThreads) { const float v = to_f32(y[c]); ss += v * v; }
        post = 1.0f / sqrtf(block_sum(ss, s_sum[0]) / (float)a.width + a.eps);
    }
    float ss = 0.f;
    uint32_t m = 0;
    for (int c = threadIdx.x; c < a.width; c += kRowThreads) {
        float v = __fmul_rn(to_f32(x[c]), a.x_scale);
        if (a.d_y) {
            float z = to_f32(y[c]);
            if (a.d_post_w) z = z * post * a.d_post_w[c];
            if (a.d_gate) z = __fmul_rn(z, gate_value(to_f32(g[c]), a.gate_kind));
            v = __fadd_rn(v, __fmul_rn(z, a.y_scale));
        }
        if (a.d_x_out) x_out[c] = from_f32<X>(v);
        ss += v * v;
        if (a.d_pre_w) v = __fmul_rn(v, a.d_pre_w[c]);
        m = max(m, q8_abs_bits(v));
        s_row[c] = v;
    }
    if (!a.d_out && !a.d_codes) return;
    const float pre = 1.0f / sqrtf(block_sum(ss, s_sum[1]) / (float)a.width + a.eps);
    if (a.d_out) {
        T* out = static_cast<T*>(a.d_out) + row * a.ld_out;
        for (int c = threadIdx.x; c < a.width; c += kRowThreads) out[c] = from_f32<T>(s_row[c] * pre);
    }
    if (a.d_codes) {
        const Q8Row q = q8_row(block_max(m, s_max));
        int8_t* codes = a.d_codes + row * a.ld_codes;
        for (int c = threadIdx.x; c < a.width; c += kRowThreads) codes[c] = (int8_t)q8_code(s_row[c], q.inv);
        if (threadIdx.x == 0) a.d_scales[row] = q.scale * pre;
    }
}

}  // namespace

int launch_q8_quantize(ElemType t, const void* x, long long ldx, int rows, int cols, int8_t* codes, long long ldc, int pad_to, float* scales, cudaStream_t s) {
    if (rows == 0) return 0;
    dispatch_elem3(t, [&](auto tag) {
        using T = decltype(tag);
        launch_pdl(q8_quantize_kernel<T>, dim3(rows), dim3(kRowThreads), 0, s, (const T*)x, ldx, cols, codes, ldc, pad_to, scales);
    });
    B2_LAUNCH_CHECK();
    return 0;
}

template <typename X, typename T>
static int norm_block(const b200attn_norm_args& a, cudaStream_t s) {
    static PerDeviceOnce once;
    B2_PER_DEVICE_ONCE(once, B2_CUDA(cudaFuncSetAttribute(norm_block_kernel<X, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormMostWidth * 4)));
    launch_pdl(norm_block_kernel<X, T>, dim3(a.rows), dim3(kRowThreads), (size_t)a.width * 4, s, a);
    B2_LAUNCH_CHECK();
    return 0;
}

int launch_norm_block(const b200attn_norm_args& a, ElemType x_type, ElemType type, cudaStream_t s) {
    if (a.rows == 0) return 0;
    int st = 0;
    dispatch_elem3(type, [&](auto tag) {
        using T = decltype(tag);
        st = x_type == ELEM_F32 ? norm_block<float, T>(a, s) : norm_block<T, T>(a, s);
    });
    return st;
}

}  // namespace b200
