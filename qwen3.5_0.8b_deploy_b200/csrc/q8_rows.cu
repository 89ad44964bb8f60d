// Row-wise kernels of the 8-bit path: the quantiser of activations, and the norm block (norms behind and in front of a block with its gate and
// residual scales, the result in 16 or 32 bits or as 8-bit codes).
//
// Both are bound by memory: every input is read once and kept in registers between the reductions over its row and the outputs that need them.  Rows of up
// to 1024 values have a warp each, without barriers; longer ones a block; those that no block's registers hold go through the two loop kernels.  Few rows get
// a thread per eight values: nothing else fills the machine then.
//   quantise 65536 x 3584 fp16                   115 us (705 MB, 108 at the copy rate; the two-pass kernel 237)
//   norm to codes, 65536 x 1024, fp32 x, fp16 y  110 us (738 MB, 113; a block per row through shared memory 299)
//   norms on both sides, 16384 x 4096, fp32 x    127 us (805 MB, 123; through shared memory 259)
// What it took beside the single pass: enough warps to cover the loads (norm to codes at 4 / 5 / 6 blocks of four warps an SM: 111.5 / 110.0 / 119.9 us, the last with
// spills; the second norm at 1 / 2 / 3 blocks: 143 / 127 / 158), and no branch on the form of the update inside the eight values of a step (130 us).
#include "elem.cuh"
#include "ptx_utils.cuh"
#include "q8.cuh"

#include <algorithm>
#include <type_traits>

namespace b200 {
namespace {

// ---- eight values of a row: side by side (kRun 8), or in pairs or one by one a block's width apart (rows that start or end off such a boundary: kRun 2
// where pairs are aligned, else 1).  777 rows of 2050 values with norms on both sides and a
// sigmoid gate: 11.9 us one by one, 9.5 in pairs (8.3 with the branches of norm_update around eight values).
template <typename T, int kRun> struct alignas(16) Raw { T v[8]; };
template <> struct alignas(16) Raw<__half, 8> { uint32_t v[4]; };
template <> struct alignas(16) Raw<__nv_bfloat16, 8> { uint32_t v[4]; };
__device__ __forceinline__ float2 unpack2(uint32_t v, __half) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
__device__ __forceinline__ float2 unpack2(uint32_t v, __nv_bfloat16) { return unpack_bf16x2(v); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) { return pack_half2(a, b); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) { return pack_bf16x2(a, b); }
__device__ __forceinline__ float2 pack2(float a, float b, float) { return make_float2(a, b); }

// Eight values in one access: 16 bytes, or 32 of fp32 values (as two of 16 bytes each lane would take half a sector at a time).  Rows pass through once and
// stay out of L1, which the weights then have for themselves.  Not through the read-only path: x may be updated in place.
__device__ __forceinline__ void load_once(const float* p, Raw<float, 8>& r) {
    float(&v)[8] = r.v;
    asm volatile("ld.global.L1::no_allocate.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(p));
}
template <typename T>
__device__ __forceinline__ void load_once(const T* p, Raw<T, 8>& r) {
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.v[0]), "=r"(r.v[1]), "=r"(r.v[2]), "=r"(r.v[3]) : "l"(p));
}

// Where a row's code of a column lies, from its first one on.
template <bool kBlocks>
__device__ __forceinline__ int code_place(int col) { return kBlocks ? col / 128 * kQ8Block + col % 128 : col; }
template <bool kBlocks>
__device__ __forceinline__ int8_t* code_row(int8_t* codes, long long row, long long pitch) {
    return codes + (kBlocks ? row / 8 * 8 * pitch + row % 8 * 128 : row * pitch);
}

template <int kRun>
struct Eight {
    int first, threads, cols;
    __device__ __forceinline__ Eight(int group, int t, int threads_, int cols_) : first(8 * group * threads_ + kRun * t), threads(threads_), cols(cols_) {}
    __device__ __forceinline__ int col(int j) const { return first + j / kRun * kRun * threads + j % kRun; }
    __device__ __forceinline__ bool any() const { return first < cols; }
    __device__ __forceinline__ bool has(int j) const { return col(j) < cols; }
    // As they come from memory, zeros behind the row.  Kernels fetch all that they need of a row before they unpack any of it.
    template <bool kOnce, typename T>
    __device__ __forceinline__ void fetch(const T* row, Raw<T, kRun>& r) const {
        if constexpr (kRun == 8) {
            if constexpr (kOnce) {
#pragma unroll
                for (auto& v : r.v) v = 0;
                if (any()) load_once(row + first, r);
            } else {
#pragma unroll
                for (int j = 0; j < (int)sizeof(T) / 2; ++j)
                    reinterpret_cast<uint4*>(&r)[j] = any() ? reinterpret_cast<const uint4*>(row + first)[j] : make_uint4(0, 0, 0, 0);
            }
        } else if constexpr (kRun == 2) {
            using P = decltype(pack2(0.f, 0.f, T{}));
#pragma unroll
            for (int j = 0; j < 8; j += 2) *reinterpret_cast<P*>(r.v + j) = has(j) ? *reinterpret_cast<const P*>(row + col(j)) : P{};
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) r.v[j] = has(j) ? row[col(j)] : T(0.f);
        }
    }
    template <typename T>
    __device__ __forceinline__ static void unpack(const Raw<T, kRun>& r, float (&v)[8]) {
        if constexpr (kRun == 8 && sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 f = unpack2(r.v[j], T{});
                v[2 * j] = f.x;
                v[2 * j + 1] = f.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = to_f32(r.v[j]);
        }
    }
    template <typename T>
    __device__ __forceinline__ void store(T* row, const float (&v)[8]) const {
        if constexpr (kRun == 8 && sizeof(T) == 4) {
            asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(row + first), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]),
                         "f"(v[6]), "f"(v[7]) : "memory");
        } else if constexpr (kRun == 8) {
            *reinterpret_cast<uint4*>(row + first) = make_uint4(pack2(v[0], v[1], T{}), pack2(v[2], v[3], T{}), pack2(v[4], v[5], T{}), pack2(v[6], v[7], T{}));
        } else if constexpr (kRun == 2) {
            using P = decltype(pack2(0.f, 0.f, T{}));
#pragma unroll
            for (int j = 0; j < 8; j += 2)
                if (has(j)) *reinterpret_cast<P*>(row + col(j)) = pack2(v[j], v[j + 1], T{});
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (has(j)) row[col(j)] = from_f32<T>(v[j]);
        }
    }
    template <bool kBlocks = false>
    __device__ __forceinline__ void store_codes(int8_t* row, const float (&v)[8], const Q8Row& q) const {
        const uint32_t lo = q8_codes4(v[0], v[1], v[2], v[3], q.inv), hi = q8_codes4(v[4], v[5], v[6], v[7], q.inv);
        if constexpr (kRun == 8) {
            *reinterpret_cast<uint2*>(row + code_place<kBlocks>(first)) = make_uint2(lo, hi);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j += kRun) {
                if (!has(j)) continue;
                const uint32_t c = (j < 4 ? lo : hi) >> (8 * (j & 3));
                if constexpr (kRun == 2) *reinterpret_cast<uint16_t*>(row + code_place<kBlocks>(col(j))) = (uint16_t)c;
                else row[code_place<kBlocks>(col(j))] = (int8_t)c;
            }
        }
    }
};

// ---- reductions over the threads of a row: a warp, or a block of up to 32 warps ---------------------------------------------------------------------
struct RowSum { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct RowMax { __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); } };
template <typename V, typename F>
__device__ __forceinline__ V warp_reduce(V v, F f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
// `part`: 32 words that nothing else uses.  Every thread returns the same value.
template <bool kWarp, typename V, typename F>
__device__ __forceinline__ V row_reduce(V v, V* part, F f) {
    v = warp_reduce(v, f);
    if constexpr (kWarp) return v;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_reduce(lane < warps ? part[lane] : V(0), f);
}

// ---- quantiser ------------------------------------------------------------------------------------------------------------------------------------------
constexpr int kBlockThreads = 512;               // most threads of a row
constexpr int kQuantGroups = 4;                  // eights of a thread
template <typename T, bool kWarp, int kRun, bool kBlocks>
__global__ void __launch_bounds__(kWarp ? 128 : kBlockThreads)
q8_quantize_kernel(const T* __restrict__ x, long long ldx, int rows, int cols, int8_t* __restrict__ codes, long long ldc, float* __restrict__ scales) {
    __shared__ uint32_t s_max[32];
    const int threads = kWarp ? 32 : blockDim.x, t = kWarp ? threadIdx.x & 31 : threadIdx.x;
    const long long row = kWarp ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    pdl_enter();
    if (row >= rows) return;
    const T* src = x + row * ldx;
    int8_t* out = code_row<kBlocks>(codes, row, ldc);
    Raw<T, kRun> raw[kQuantGroups];
#pragma unroll
    for (int i = 0; i < kQuantGroups; ++i) Eight<kRun>(i, t, threads, cols).template fetch<true>(src, raw[i]);
    uint32_t m = 0;
    float v[8];
#pragma unroll
    for (int i = 0; i < kQuantGroups; ++i) {
        const uint32_t* words = reinterpret_cast<const uint32_t*>(raw[i].v);
#pragma unroll
        for (int j = 0; j < 2 * (int)sizeof(T); ++j) m = q8_max_word<T>(m, words[j]);
    }
    m = q8_max_bits<T>(m);
    const Q8Row q = q8_row(row_reduce<kWarp>(m, s_max, RowMax{}));
#pragma unroll
    for (int i = 0; i < kQuantGroups; ++i) {
        const Eight<kRun> e(i, t, threads, cols);
        if (!e.any()) break;
        Eight<kRun>::unpack(raw[i], v);
        e.template store_codes<kBlocks>(out, v, q);
    }
    if constexpr (kBlocks)
        for (int c = cols + t; c < ldc; c += threads) out[code_place<true>(c)] = 0;
    if (t == 0) scales[row] = q.scale;
}

// A block per row, two passes over it.
constexpr int kLoopThreads = kBlockThreads;
template <typename T, bool kBlocks>
__global__ void __launch_bounds__(kLoopThreads)
q8_quantize_loop_kernel(const T* __restrict__ x, long long ldx, int cols, int8_t* __restrict__ codes, long long ldc, float* __restrict__ scales) {
    __shared__ uint32_t s_max[32];
    pdl_enter();
    const T* row = x + blockIdx.x * ldx;
    int8_t* out = code_row<kBlocks>(codes, blockIdx.x, ldc);
    uint32_t m = 0;
    for (int c = threadIdx.x; c < cols; c += kLoopThreads) m = max(m, q8_abs_bits(to_f32(row[c])));
    const Q8Row q = q8_row(row_reduce<false>(m, s_max, RowMax{}));
    for (int c = threadIdx.x; c < cols; c += kLoopThreads) out[code_place<kBlocks>(c)] = (int8_t)q8_code(to_f32(row[c]), q.inv);
    if constexpr (kBlocks)
        for (int c = cols + threadIdx.x; c < ldc; c += kLoopThreads) out[code_place<true>(c)] = 0;
    if (threadIdx.x == 0) scales[blockIdx.x] = q.scale;
}

__global__ void __launch_bounds__(256)
q8_unblock_kernel(const int8_t* __restrict__ codes, int pitch, int cols, int8_t* __restrict__ out) {
    pdl_enter();
    for (int c = threadIdx.x; c < cols; c += 256) out[(size_t)blockIdx.x * cols + c] = codes[q8_block_offset(blockIdx.x, c, pitch)];
}

// ---- norm block -----------------------------------------------------------------------------------------------------------------------------------------
// x' of N values, in place of x: products and sums are rounded one by one, so that the codes are what the formula gives in 32 bits, whatever contracts there.
template <int N>
__device__ __forceinline__ void norm_update(const b200attn_norm_args& a, float (&x)[N], float (&y)[N], float post, const float (&post_w)[N], const float (&gate)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = __fmul_rn(x[j], a.x_scale);
    if (!a.d_y) return;
    if (a.d_post_w) {
#pragma unroll
        for (int j = 0; j < N; ++j) y[j] = y[j] * post * post_w[j];
    }
    if (a.d_gate) {
        if (a.gate_kind == B200ATTN_GATE_SIGMOID) {
#pragma unroll
            for (int j = 0; j < N; ++j) y[j] = y[j] * (1.0f / (1.0f + expf(-gate[j])));
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) y[j] = __fmul_rn(y[j], gate[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = __fadd_rn(x[j], __fmul_rn(y[j], a.y_scale));
}
__device__ __forceinline__ float norm_rms(float squares, const b200attn_norm_args& a) { return sqrtf(squares / (float)a.width + a.eps); }

template <typename X, typename T, int kGroups, bool kWarp, int kRun>
__global__ void __launch_bounds__(kWarp ? 128 : kBlockThreads, kRun < 8 ? 1 : kWarp ? 5 : kGroups > 2 ? 1 : 2)
norm_block_kernel(const b200attn_norm_args a) {
    __shared__ float s_post[32], s_pre[32];
    __shared__ uint32_t s_max[32];
    const int threads = kWarp ? 32 : blockDim.x, t = kWarp ? threadIdx.x & 31 : threadIdx.x;
    const long long row = kWarp ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    pdl_enter();
    if (row >= a.rows) return;
    const X* x = static_cast<const X*>(a.d_x) + row * a.ldx;
    const T* y = static_cast<const T*>(a.d_y) + row * a.ldy;
    const T* g = static_cast<const T*>(a.d_gate) + row * a.ld_gate;
    using E = Eight<kRun>;
    Raw<X, kRun> rx[kGroups];
    Raw<T, kRun> ry[kGroups], rg[kGroups];
    Raw<float, kRun> rw[2];                      // weights of a single group come with the rest, those of more when they are wanted
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const E e(i, t, threads, a.width);
        if (a.d_y) e.template fetch<true>(y, ry[i]);
        e.template fetch<true>(x, rx[i]);
        if (a.d_gate) {
            if (a.ld_gate) e.template fetch<true>(g, rg[i]);
            else e.template fetch<false>(g, rg[i]);
        }
        if (kGroups == 1 && a.d_post_w) e.template fetch<false>(a.d_post_w, rw[0]);
        if (kGroups == 1 && a.d_pre_w) e.template fetch<false>(a.d_pre_w, rw[1]);
    }
    float v[kGroups][8], z[8], gate[8], w[8];
    float post = 1.f, ss = 0.f;
    if (a.d_post_w) {
#pragma unroll
        for (int i = 0; i < kGroups; ++i) {
            E::unpack(ry[i], z);
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += z[j] * z[j];
        }
        post = 1.0f / norm_rms(row_reduce<kWarp>(ss, s_post, RowSum{}), a);
        ss = 0.f;
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const E e(i, t, threads, a.width);
        if (!e.any()) break;
        E::unpack(rx[i], v[i]);
        E::unpack(ry[i], z);
        E::unpack(rg[i], gate);
        if (a.d_post_w) {
            if (kGroups > 1) e.template fetch<false>(a.d_post_w, rw[0]);
            E::unpack(rw[0], w);
        }
        norm_update(a, v[i], z, post, w, gate);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += v[i][j] * v[i][j];           // zeros stay zeros
        if (a.d_x_out) e.store(static_cast<X*>(a.d_x_out) + row * a.ldx_out, v[i]);
        if (a.d_pre_w) {
            if (kGroups > 1) e.template fetch<false>(a.d_pre_w, rw[1]);
            E::unpack(rw[1], w);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = __fmul_rn(v[i][j], w[j]);
        }
        if (a.d_codes) {
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, q8_abs_bits(v[i][j]));
        }
    }
    if (!a.d_out && !a.d_codes) return;
    const float rms = norm_rms(row_reduce<kWarp>(ss, s_pre, RowSum{}), a), pre = 1.0f / rms;
    Q8Row q{};
    if (a.d_codes) {
        q = q8_row(row_reduce<kWarp>(m, s_max, RowMax{}));
        if (t == 0) a.d_scales[row] = q.scale / rms;
    }
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const E e(i, t, threads, a.width);
        if (!e.any()) break;
        if (a.d_codes) e.store_codes(a.d_codes + row * a.ld_codes, v[i], q);
        if (a.d_out) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] *= pre;
            e.store(static_cast<T*>(a.d_out) + row * a.ld_out, v[i]);
        }
    }
}

// A block per row, the updated row in shared memory between the passes.
template <typename X, typename T>
__global__ void __launch_bounds__(kLoopThreads)
norm_block_loop_kernel(const b200attn_norm_args a) {
    extern __shared__ float s_row[];
    __shared__ float s_post[32], s_pre[32];
    __shared__ uint32_t s_max[32];
    pdl_enter();
    const long long row = blockIdx.x;
    const X* x = static_cast<const X*>(a.d_x) + row * a.ldx;
    const T* y = static_cast<const T*>(a.d_y) + row * a.ldy;
    const T* g = static_cast<const T*>(a.d_gate) + row * a.ld_gate;
    X* x_out = static_cast<X*>(a.d_x_out) + row * a.ldx_out;
    float post = 1.f;
    if (a.d_post_w) {
        float ss = 0.f;
        for (int c = threadIdx.x; c < a.width; c += kLoopThreads) { const float v = to_f32(y[c]); ss += v * v; }
        post = 1.0f / norm_rms(row_reduce<false>(ss, s_post, RowSum{}), a);
    }
    float ss = 0.f;
    uint32_t m = 0;
    for (int c = threadIdx.x; c < a.width; c += kLoopThreads) {
        float u[1] = {to_f32(x[c])}, z[1] = {a.d_y ? to_f32(y[c]) : 0.f};
        const float w[1] = {a.d_post_w ? a.d_post_w[c] : 1.f}, gate[1] = {a.d_gate ? to_f32(g[c]) : 1.f};
        norm_update(a, u, z, post, w, gate);
        float v = u[0];
        if (a.d_x_out) x_out[c] = from_f32<X>(v);
        ss += v * v;
        if (a.d_pre_w) v = __fmul_rn(v, a.d_pre_w[c]);
        m = max(m, q8_abs_bits(v));
        s_row[c] = v;
    }
    if (!a.d_out && !a.d_codes) return;
    const float rms = norm_rms(row_reduce<false>(ss, s_pre, RowSum{}), a), pre = 1.0f / rms;
    if (a.d_out) {
        T* out = static_cast<T*>(a.d_out) + row * a.ld_out;
        for (int c = threadIdx.x; c < a.width; c += kLoopThreads) out[c] = from_f32<T>(s_row[c] * pre);
    }
    if (a.d_codes) {
        const Q8Row q = q8_row(row_reduce<false>(m, s_max, RowMax{}));
        int8_t* codes = a.d_codes + row * a.ld_codes;
        for (int c = threadIdx.x; c < a.width; c += kLoopThreads) codes[c] = (int8_t)q8_code(s_row[c], q.inv);
        if (threadIdx.x == 0) a.d_scales[row] = q.scale / rms;
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------------------------------
// How many values of rows [.., ld] lie side by side on a boundary of their own, so that they are one access: 8, 2 or 1.
int run_of(int cols, const void* p, long long ld, size_t bytes) {
    for (const int run : {8, 2}) {
        const size_t access = run * bytes;
        if (cols % run == 0 && reinterpret_cast<uintptr_t>(p) % access == 0 && ld * bytes % access == 0) return run;
    }
    return 1;
}
template <typename F>
void dispatch_run(int run, F&& f) {
    if (run == 8) f(std::integral_constant<int, 8>{});
    else if (run == 2) f(std::integral_constant<int, 2>{});
    else f(std::integral_constant<int, 1>{});
}
int threads_for(int cols, int groups) { return std::max(64, (ceil_div(cols, 8 * groups) + 31) / 32 * 32); }

template <bool kBlocks>
int quantize(ElemType t, const void* x, long long ldx, int rows, int cols, int8_t* codes, long long ldc, float* scales, cudaStream_t s) {
    if (rows == 0) return 0;
    dispatch_elem3(t, [&](auto tag) {
        using T = decltype(tag);
        const T* src = static_cast<const T*>(x);
        dispatch_run(std::min(run_of(cols, x, ldx, sizeof(T)), run_of(cols, codes, ldc, 1)), [&](auto run) {
            constexpr int kRun = decltype(run)::value;
            if (cols <= 32 * 8 * kQuantGroups)
                launch_pdl(q8_quantize_kernel<T, true, kRun, kBlocks>, dim3(ceil_div(rows, 4)), dim3(128), 0, s, src, ldx, rows, cols, codes, ldc, scales);
            else if (cols <= kBlockThreads * 8 * kQuantGroups)
                launch_pdl(q8_quantize_kernel<T, false, kRun, kBlocks>, dim3(rows), dim3(threads_for(cols, kQuantGroups)), 0, s, src, ldx, rows, cols, codes, ldc, scales);
            else
                launch_pdl(q8_quantize_loop_kernel<T, kBlocks>, dim3(rows), dim3(kLoopThreads), 0, s, src, ldx, cols, codes, ldc, scales);
        });
    });
    B2_LAUNCH_CHECK();
    return 0;
}

template <typename X, typename T, int kRun>
int norm_block(const b200attn_norm_args& a, cudaStream_t s) {
    const auto wide = [&](auto kernel, int groups) { launch_pdl(kernel, dim3(a.rows), dim3(threads_for(a.width, groups)), 0, s, a); };
    // A thread per eight values as long as all rows are under way at once with them (64 registers each), else fewer threads that have more to wait for: 1000 x 4096
    // 10.3 us, with 512 threads a row 13.5.  Values one by one or in pairs keep more threads busy: 777 x 2050 8.4 us, with two eights a thread 10.4.
    int sms = 0;
    B2_TRY(device_sm_count(&sms));
    const int few = kRun == 8 ? sms * (1024 / threads_for(a.width, 1)) : 1024;
    if (a.width <= 4096 && a.rows <= few) wide(norm_block_kernel<X, T, 1, false, kRun>, 1);
    else if (a.width <= 1024) launch_pdl(norm_block_kernel<X, T, 4, true, kRun>, dim3(ceil_div(a.rows, 4)), dim3(128), 0, s, a);
    else if (a.width <= 8192) wide(norm_block_kernel<X, T, 2, false, kRun>, 2);
    else if (a.width <= 16384) wide(norm_block_kernel<X, T, 4, false, kRun>, 4);
    else {
        static PerDeviceOnce once;
        B2_PER_DEVICE_ONCE(once, B2_CUDA(cudaFuncSetAttribute(norm_block_loop_kernel<X, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormMostWidth * 4)));
        launch_pdl(norm_block_loop_kernel<X, T>, dim3(a.rows), dim3(kLoopThreads), (size_t)a.width * 4, s, a);
    }
    B2_LAUNCH_CHECK();
    return 0;
}

}  // namespace

int launch_q8_quantize(ElemType t, const void* x, long long ldx, int rows, int cols, int8_t* codes, long long ldc, float* scales, cudaStream_t s) {
    return quantize<false>(t, x, ldx, rows, cols, codes, ldc, scales, s);
}
int launch_q8_quantize_weights(ElemType t, const void* w, long long ldw, int rows, int cols, int8_t* codes, int pitch, float* scales, cudaStream_t s) {
    return quantize<true>(t, w, ldw, rows, cols, codes, pitch, scales, s);
}

int launch_q8_unblock(const int8_t* codes, int pitch, int rows, int cols, int8_t* out, cudaStream_t s) {
    launch_pdl(q8_unblock_kernel, dim3(rows), dim3(256), 0, s, codes, pitch, cols, out);
    B2_LAUNCH_CHECK();
    return 0;
}

int launch_norm_block(const b200attn_norm_args& a, ElemType x_type, ElemType type, cudaStream_t s) {
    const size_t xb = elem_bytes(x_type), b = elem_bytes(type);
    int run = 8, st = 0;
    auto with = [&](const void* p, long long ld, size_t bytes) { run = std::min(run, run_of(a.width, p, ld, bytes)); };
    with(a.d_x, a.ldx, xb);
    if (a.d_x_out) with(a.d_x_out, a.ldx_out, xb);
    if (a.d_y) with(a.d_y, a.ldy, b);
    if (a.d_gate) with(a.d_gate, a.ld_gate, b);
    if (a.d_out) with(a.d_out, a.ld_out, b);
    if (a.d_codes) with(a.d_codes, a.ld_codes, 1);
    if (a.d_post_w) with(a.d_post_w, 0, 4);
    if (a.d_pre_w) with(a.d_pre_w, 0, 4);
    dispatch_elem3(type, [&](auto tag) {
        using T = decltype(tag);
        dispatch_run(run, [&](auto r) {
            constexpr int kRun = decltype(r)::value;
            st = x_type == ELEM_F32 ? norm_block<float, T, kRun>(a, s) : norm_block<T, T, kRun>(a, s);
        });
    });
    return st;
}

}  // namespace b200
