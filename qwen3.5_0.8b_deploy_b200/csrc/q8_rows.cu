// Row-wise kernels of the 8-bit path: the quantiser of activations, and the norm block (norms behind and in front of a block with its gate and
// residual scales, the result in 16 or 32 bits or as 8-bit codes).
//
// Both are bound by memory: every input is read once and kept in registers between the reductions over its row and the outputs that need them.  Short rows have
// some lanes of a warp each, without barriers, so that a warp holds several; longer ones a block; those that no block's registers hold go through the two loop kernels.
//   quantise 65536 x 3584 fp16                   102 us (705 MB, 108 at the copy rate; the two-pass kernel 237)
//   quantise 65536 x 256 bf16                    6.4 us from L2 (a warp per row 17.7)
//   norm to codes, 65536 x 1024, fp32 x, fp16 y  111 us (738 MB, 113; a block per row through shared memory 299)
//   norms on both sides, 16384 x 4096, fp32 x    127 us (805 MB, 123; through shared memory 259)
//   norms on both sides, 49268 x 64, fp32 x      6.5 us from L2 (a warp per row 28.4)
// What it took beside the single pass: enough warps to cover the loads (norm to codes at 4 / 5 / 6 blocks of four warps an SM: 111.5 / 110.0 / 119.9 us, the last with
// spills; the second norm at 1 / 2 / 3 blocks: 143 / 127 / 158), no branch on the form of the update inside the eight values of a step (130 us), and a largest value
// found in packed pairs (the quantiser 115 us without).  All in fp32, norm blocks of 520 to 1024 columns spill 80 bytes a thread at five blocks: 65536 x 1024 164 us, with a
// norm behind the block 171 (164 at the copy rate).  Rows of an odd width are bound by their instructions: 30000 x 2501 bf16 to codes 48 us, 34 at the copy rate.
#include "elem.cuh"
#include "ptx_utils.cuh"
#include "q8.cuh"

#include <algorithm>
#include <type_traits>

namespace b200 {
namespace {

// ---- eight values of a row ----------------------------------------------------------------------------------------------------------------------------------
// kEights: side by side from a multiple of eight on, all rows on boundaries of eight values.  The other rows:
// kSingles: one by one, a row's threads apart.  The threads are a constant there, so that the eight addresses differ by constants.
// kShifted: a block's rows that all lie alike against such boundaries (rows of an odd width do): a thread's eight begin as many columns earlier as the row begins
// behind a boundary, so that they are one access again; weights and codes, which lie otherwise, are turned into place in registers.  What that takes pays for rows above
// 1024 values: 10000 x 15001 bf16 to codes 90 us, one by one 185; 30000 x 2501 50, 62; but 39816 x 771 24, 22; norms of 5000 x 3001 57, 91; 3000 x 700 8.7, 7.9.
enum { kSingles = 1, kEights = 8, kShifted = 9 };
constexpr int kFewestShifted = 1025;             // columns
template <typename T, bool kWords> struct alignas(16) RawEight { T v[8]; };
template <> struct alignas(16) RawEight<__half, true> { uint32_t v[4]; };
template <> struct alignas(16) RawEight<__nv_bfloat16, true> { uint32_t v[4]; };
template <typename T, int kRun> using Raw = RawEight<T, kRun != kSingles>;
__device__ __forceinline__ float2 unpack2(uint32_t v, __half) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
__device__ __forceinline__ float2 unpack2(uint32_t v, __nv_bfloat16) { return unpack_bf16x2(v); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) { return pack_half2(a, b); }
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) { return pack_bf16x2(a, b); }

// Eight values in one access: 16 bytes, or 32 of fp32 values (as two of 16 bytes each lane would take half a sector at a time).  Rows pass through once and
// stay out of L1, which the weights then have for themselves.  Not through the read-only path: x may be updated in place.
__device__ __forceinline__ void load_once(const float* p, float (&v)[8]) {
    asm volatile("ld.global.L1::no_allocate.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]) : "l"(p));
}
template <typename T>
__device__ __forceinline__ void load_once(const T* p, uint32_t (&v)[4]) {
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "l"(p));
}

// Where a row's code of a column lies, from its first one on.
template <bool kBlocks>
__device__ __forceinline__ int code_place(int col) { return kBlocks ? col / 128 * kQ8Block + col % 128 : col; }
template <bool kBlocks>
__device__ __forceinline__ int8_t* code_row(int8_t* codes, long long row, long long pitch) {
    return codes + (kBlocks ? row / 8 * 8 * pitch + row % 8 * 128 : row * pitch);
}

// kThreads: of a row, 0: as many as the block has.
template <int kThreads>
__device__ __forceinline__ int row_threads() { return kThreads ? kThreads : blockDim.x; }

// Where a row lies (kShifted): values from the last boundary of eight to its first one, and values of the same matrix in front of the row and behind it, if less than 8.
struct Place {
    int shift = 0, before = 0, after = 0;
};
template <int kRun, typename T>
__device__ __forceinline__ Place place_of(const T* ptr, long long row, long long rows) {
    if constexpr (kRun != kShifted) return {};
    return {(int)(reinterpret_cast<uintptr_t>(ptr) / sizeof(T) % 8), row > 0 ? 8 : 0, row + 1 < rows ? 8 : 0};
}

template <int kRun, int kThreads>
struct Eight {
    int first, cols;
    Place place;
    __device__ __forceinline__ Eight(int group, int t, int cols_, const Place& place_)
        : first(8 * group * row_threads<kThreads>() + (kRun == kSingles ? t : 8 * t - place_.shift)), cols(cols_), place(place_) {}
    __device__ __forceinline__ int col(int j) const { return first + (kRun == kSingles ? j * row_threads<kThreads>() : j); }
    __device__ __forceinline__ bool any() const { return first < cols; }
    __device__ __forceinline__ bool has(int j) const { return kRun == kShifted ? (unsigned)col(j) < (unsigned)cols : col(j) < cols; }
    __device__ __forceinline__ bool whole() const { return first >= 0 && first + 8 <= cols; }
    template <typename T>
    __device__ __forceinline__ void fetch_each(const T* row, Raw<T, kRun>& r) const {
        if constexpr (sizeof(T) == 2 && kRun != kSingles) {
            const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                r.v[j] = (has(2 * j) ? (uint32_t)p[col(2 * j)] : 0u) | (has(2 * j + 1) ? (uint32_t)p[col(2 * j + 1)] << 16 : 0u);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) r.v[j] = has(j) ? row[col(j)] : T(0.f);
        }
    }
    // As they come from memory, zeros outside the row (kShifted: behind `trim`).  Kernels fetch all that they need of a row before they unpack any of it.
    template <typename T>
    __device__ __forceinline__ void fetch(const T* row, Raw<T, kRun>& r) const {
        if constexpr (kRun == kSingles) {
            fetch_each(row, r);
        } else {
#pragma unroll
            for (auto& v : r.v) v = 0;
            if (any() && (kRun == kEights || (first >= -place.before && first <= cols - 8 + place.after))) load_once(row + first, r.v);
            else if (kRun == kShifted && any()) fetch_each(row, r);                  // the first or the last values of the matrix
        }
    }
    // Zeros in place of the neighbours' values.  Once everything has been asked for: it waits for the values.
    template <typename T>
    __device__ __forceinline__ void trim(Raw<T, kRun>& r) const {
        if constexpr (kRun == kShifted) {
            if (whole()) return;
#pragma unroll
            for (int j = 0; j < 8; j += 8 / (2 * (int)sizeof(T))) {
                if constexpr (sizeof(T) == 4) r.v[j] = has(j) ? r.v[j] : 0.f;
                else r.v[j / 2] &= (has(j) ? 0xffffu : 0u) | (has(j + 1) ? 0xffff0000u : 0u);
            }
        }
    }
    // Of a vector that all rows share.
    template <typename T>
    __device__ __forceinline__ void fetch_shared(const T* vec, Raw<T, kRun>& r) const {
        if constexpr (kRun == kEights) {
#pragma unroll
            for (int j = 0; j < (int)sizeof(T) / 2; ++j)
                reinterpret_cast<uint4*>(&r)[j] = any() ? reinterpret_cast<const uint4*>(vec + first)[j] : make_uint4(0, 0, 0, 0);
        } else if constexpr (kRun == kShifted && sizeof(T) == 4) {
            const int off = (int)(reinterpret_cast<uintptr_t>(vec + first) / 4 % 4);            // the same for all threads of a row
            const bool inside = first >= off && first - off + 12 <= cols;
            float q[12];
#pragma unroll
            for (int j = 0; j < 12; j += 4) {
                const int c = first - off + j;
                float4& f = *reinterpret_cast<float4*>(q + j);
                if (inside || (c >= 0 && c + 4 <= cols)) {
                    f = *reinterpret_cast<const float4*>(vec + c);
                } else {
                    f.x = c >= 0 && c < cols ? vec[c] : 0.f;
                    f.y = c >= -1 && c + 1 < cols ? vec[c + 1] : 0.f;
                    f.z = c >= -2 && c + 2 < cols ? vec[c + 2] : 0.f;
                    f.w = c >= -3 && c + 3 < cols ? vec[c + 3] : 0.f;
                }
            }
#pragma unroll
            for (int j = 0; j < 10; ++j) q[j] = off & 2 ? q[j + 2] : q[j];
#pragma unroll
            for (int j = 0; j < 8; ++j) r.v[j] = off & 1 ? q[j + 1] : q[j];
        } else {
            fetch_each(vec, r);
        }
    }
    template <typename T>
    __device__ __forceinline__ static void unpack(const Raw<T, kRun>& r, float (&v)[8]) {
        if constexpr (kRun != kSingles && sizeof(T) == 2) {
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
        if (kRun == kEights || (kRun == kShifted && whole())) {
            if constexpr (sizeof(T) == 4)
                asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(row + first), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]),
                             "f"(v[6]), "f"(v[7]) : "memory");
            else
                *reinterpret_cast<uint4*>(row + first) = make_uint4(pack2(v[0], v[1], T{}), pack2(v[2], v[3], T{}), pack2(v[4], v[5], T{}), pack2(v[6], v[7], T{}));
        } else if constexpr (kRun != kEights) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (has(j)) row[col(j)] = from_f32<T>(v[j]);
        }
    }
    // Eight codes (lo, hi).  kShifted: those from the multiple of eight columns on that lies in this thread's eight values (exchange).
    template <bool kBlocks = false>
    __device__ __forceinline__ void store_codes(int8_t* row, uint32_t lo, uint32_t hi) const {
        if constexpr (kRun == kEights) {
            *reinterpret_cast<uint2*>(row + code_place<kBlocks>(first)) = make_uint2(lo, hi);
        } else if constexpr (kRun == kSingles) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (has(j)) row[code_place<kBlocks>(col(j))] = (int8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
        } else {
            const int c = first + place.shift, n = cols - c;
            int8_t* dst = row + code_place<kBlocks>(c);
            if (reinterpret_cast<uintptr_t>(row) % 8 == 0) {
                if (n >= 8) {
                    *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
                } else if (n > 0) {
                    if (n & 4) *reinterpret_cast<uint32_t*>(dst) = lo;
                    uint32_t rest = n & 4 ? hi : lo;
                    dst += n & 4;
                    if (n & 2) { *reinterpret_cast<uint16_t*>(dst) = (uint16_t)rest; rest >>= 16; }
                    if (n & 1) dst[n & 2] = (int8_t)rest;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < n) dst[j] = (int8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
            }
        }
    }
};
__device__ __forceinline__ void codes8(const float (&v)[8], const Q8Row& q, uint32_t& lo, uint32_t& hi) {
    lo = q8_codes4(v[0], v[1], v[2], v[3], q.inv);
    hi = q8_codes4(v[4], v[5], v[6], v[7], q.inv);
}

// kShifted: in place of a thread's eight codes of each group those from the next multiple of eight columns on, the first of which are this thread's, the others of the
// thread behind it.  The first lane of a warp leaves its codes for the last one of the warp in front; the last thread's pass the end of the row.  For all threads of a block.
template <int kGroups>
__device__ __forceinline__ void exchange(uint32_t (&lo)[kGroups], uint32_t (&hi)[kGroups], int shift, uint2* heads) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < kGroups; ++i) heads[i * warps + warp] = make_uint2(lo[i], hi[i]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        uint2 next = make_uint2(__shfl_down_sync(0xffffffffu, lo[i], 1), __shfl_down_sync(0xffffffffu, hi[i], 1));
        if (lane == 31 && i * warps + warp + 1 < kGroups * warps) next = heads[i * warps + warp + 1];
        const bool far = shift >= 4;
        const uint32_t w0 = far ? hi[i] : lo[i], w1 = far ? next.x : hi[i], w2 = far ? next.y : next.x;
        lo[i] = __funnelshift_r(w0, w1, 8 * shift);          // modulo 32
        hi[i] = __funnelshift_r(w1, w2, 8 * shift);
    }
}

// ---- reductions over the threads of a row: lanes of a warp, or a block of up to 32 warps ---------------------------------------------------------------------
struct RowSum { __device__ __forceinline__ float operator()(float a, float b) const { return a + b; } };
struct RowMax { __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return max(a, b); } };
template <typename V, typename F>
__device__ __forceinline__ V warp_reduce(V v, F f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
// `part`: 32 words that nothing else uses.  Every thread of the row returns the same value.  kThreads: a power of two up to 32, or those of a block.
template <int kThreads, typename V, typename F>
__device__ __forceinline__ V row_reduce(V v, V* part, F f) {
    if constexpr (kThreads > 0 && kThreads <= 32) {
#pragma unroll
        for (int o = kThreads / 2; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    }
    v = warp_reduce(v, f);
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_reduce(lane < warps ? part[lane] : V(0), f);
}

// ---- quantiser ------------------------------------------------------------------------------------------------------------------------------------------
constexpr int kBlockThreads = 512;               // most threads of a row
constexpr int kQuantGroups = 4;                  // eights of a thread
// The threads of a row: kThreads lanes of a warp (blocks of kLaneThreads then hold several rows), or a block.
constexpr int kLaneThreads = 128;
constexpr bool in_lanes(int threads) { return threads > 0 && threads <= 32; }
template <int kThreads>
__device__ __forceinline__ long long row_of() {
    return in_lanes(kThreads) ? (long long)blockIdx.x * (kLaneThreads / kThreads) + threadIdx.x / kThreads : blockIdx.x;
}
template <int kThreads>
__device__ __forceinline__ int thread_of() { return in_lanes(kThreads) ? threadIdx.x % kThreads : threadIdx.x; }

template <typename T, int kRun, int kThreads, int kGroups, bool kBlocks>
__global__ void __launch_bounds__(in_lanes(kThreads) ? kLaneThreads : kThreads ? kThreads : kBlockThreads)
q8_quantize_kernel(const T* __restrict__ x, long long ldx, int rows, int cols, int8_t* __restrict__ codes, long long ldc, float* __restrict__ scales) {
    __shared__ uint32_t s_max[32];
    __shared__ uint2 s_heads[kRun == kShifted ? kGroups * kBlockThreads / 32 : 1];
    using E = Eight<kRun, kThreads>;
    const int t = thread_of<kThreads>();
    const long long row = row_of<kThreads>();
    pdl_enter();
    const bool live = row < rows;                // the lanes of a warp stay together
    const T* src = x + row * ldx;
    int8_t* out = code_row<kBlocks>(codes, row, ldc);
    const int width = live ? cols : 0;
    const Place place = place_of<kRun>(src, row, rows);
    Raw<T, kRun> raw[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) E(i, t, width, place).fetch(src, raw[i]);
    uint32_t m = 0;
    float v[8];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        E(i, t, width, place).trim(raw[i]);
        const uint32_t* words = reinterpret_cast<const uint32_t*>(raw[i].v);
#pragma unroll
        for (int j = 0; j < 2 * (int)sizeof(T); ++j) m = q8_max_word<T>(m, words[j]);
    }
    m = q8_max_bits<T>(m);
    const Q8Row q = q8_row(row_reduce<kThreads>(m, s_max, RowMax{}));
    uint32_t lo[kGroups], hi[kGroups];
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const E e(i, t, width, place);
        if (kRun != kShifted && !e.any()) break;
        E::unpack(raw[i], v);
        codes8(v, q, lo[i], hi[i]);
        if constexpr (kRun != kShifted) e.template store_codes<kBlocks>(out, lo[i], hi[i]);
    }
    if constexpr (kRun == kShifted) {
        exchange(lo, hi, place.shift, s_heads);
#pragma unroll
        for (int i = 0; i < kGroups; ++i) E(i, t, width, place).template store_codes<kBlocks>(out, lo[i], hi[i]);
    }
    if (!live) return;
    if constexpr (kBlocks)
        for (int c = cols + t; c < ldc; c += row_threads<kThreads>()) out[code_place<true>(c)] = 0;
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
    const Q8Row q = q8_row(row_reduce<0>(m, s_max, RowMax{}));
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

template <typename X, typename T, int kRun, int kThreads, int kGroups>
__global__ void __launch_bounds__(in_lanes(kThreads) ? kLaneThreads : kThreads ? kThreads : kBlockThreads,
                                  kRun == kSingles ? 1 : in_lanes(kThreads) ? (kGroups == 1 ? 8 : 5) : kGroups > (kRun == kEights ? 2 : 1) ? 1 : 2)
norm_block_kernel(const b200attn_norm_args a) {
    __shared__ float s_post[32], s_pre[32];
    __shared__ uint32_t s_max[32];
    __shared__ uint2 s_heads[kRun == kShifted ? kGroups * kBlockThreads / 32 : 1];
    using E = Eight<kRun, kThreads>;
    const int t = thread_of<kThreads>();
    const long long row = row_of<kThreads>();
    pdl_enter();
    const bool live = row < a.rows;              // the lanes of a warp stay together
    const int width = live ? a.width : 0;
    const X* x = static_cast<const X*>(a.d_x) + row * a.ldx;
    const T* y = static_cast<const T*>(a.d_y) + row * a.ldy;
    const T* g = static_cast<const T*>(a.d_gate) + row * a.ld_gate;
    const Place place = place_of<kRun>(x, row, a.rows);
    Raw<X, kRun> rx[kGroups];
    Raw<T, kRun> ry[kGroups], rg[kGroups];
    Raw<float, kRun> rw[2];                      // weights of a single group come with the rest, those of more when they are wanted
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const E e(i, t, width, place);
        if (a.d_y) e.fetch(y, ry[i]);
        e.fetch(x, rx[i]);
        if (a.d_gate) {
            if (a.ld_gate) e.fetch(g, rg[i]);
            else e.fetch_shared(g, rg[i]);
        }
        if (kGroups == 1 && a.d_post_w) e.fetch_shared(a.d_post_w, rw[0]);
        if (kGroups == 1 && a.d_pre_w) e.fetch_shared(a.d_pre_w, rw[1]);
    }
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const E e(i, t, width, place);
        e.trim(rx[i]);
        if (a.d_y) e.trim(ry[i]);
        if (a.d_gate) e.trim(rg[i]);
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
        post = 1.0f / norm_rms(row_reduce<kThreads>(ss, s_post, RowSum{}), a);
        ss = 0.f;
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const E e(i, t, width, place);
        if (!e.any()) {
            if (kRun != kShifted) break;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.f;               // codes of zeros are handed to the thread in front
            continue;
        }
        E::unpack(rx[i], v[i]);
        E::unpack(ry[i], z);
        E::unpack(rg[i], gate);
        if (a.d_post_w) {
            if (kGroups > 1) e.fetch_shared(a.d_post_w, rw[0]);
            E::unpack(rw[0], w);
        }
        norm_update(a, v[i], z, post, w, gate);
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += v[i][j] * v[i][j];           // zeros stay zeros
        if (a.d_x_out) e.store(static_cast<X*>(a.d_x_out) + row * a.ldx_out, v[i]);
        if (a.d_pre_w) {
            if (kGroups > 1) e.fetch_shared(a.d_pre_w, rw[1]);
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
    const float rms = norm_rms(row_reduce<kThreads>(ss, s_pre, RowSum{}), a), pre = 1.0f / rms;
    Q8Row q{};
    uint32_t lo[kGroups], hi[kGroups];
    if (a.d_codes) {
        q = q8_row(row_reduce<kThreads>(m, s_max, RowMax{}));
        if (live && t == 0) a.d_scales[row] = q.scale / rms;
        if constexpr (kRun == kShifted) {
#pragma unroll
            for (int i = 0; i < kGroups; ++i) codes8(v[i], q, lo[i], hi[i]);
            exchange(lo, hi, place.shift, s_heads);
        }
    }
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
        const E e(i, t, width, place);
        if (!e.any()) break;
        if (a.d_codes) {
            if constexpr (kRun != kShifted) codes8(v[i], q, lo[i], hi[i]);
            e.store_codes(a.d_codes + row * a.ld_codes, lo[i], hi[i]);
        }
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
        post = 1.0f / norm_rms(row_reduce<0>(ss, s_post, RowSum{}), a);
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
    const float rms = norm_rms(row_reduce<0>(ss, s_pre, RowSum{}), a), pre = 1.0f / rms;
    if (a.d_out) {
        T* out = static_cast<T*>(a.d_out) + row * a.ld_out;
        for (int c = threadIdx.x; c < a.width; c += kLoopThreads) out[c] = from_f32<T>(s_row[c] * pre);
    }
    if (a.d_codes) {
        const Q8Row q = q8_row(row_reduce<0>(m, s_max, RowMax{}));
        int8_t* codes = a.d_codes + row * a.ld_codes;
        for (int c = threadIdx.x; c < a.width; c += kLoopThreads) codes[c] = (int8_t)q8_code(s_row[c], q.inv);
        if (threadIdx.x == 0) a.d_scales[row] = q.scale / rms;
    }
}

// ---- launches -------------------------------------------------------------------------------------------------------------------------------------------
// How the rows of a call's matrices lie against boundaries of eight values.
struct Rows {
    int first = -1, step = 0;        // values behind such a boundary, and how many more from one row to the next
    bool alike = true;
    void add(const void* p, long long ld, size_t bytes) {
        const int f = (int)(reinterpret_cast<uintptr_t>(p) / bytes % 8), s = (int)(ld % 8);
        if (first < 0) { first = f; step = s; }
        alike = alike && f == first && s == step;
    }
    // others: whether codes and what rows share lie on such boundaries too
    int run(int width, bool others) const {
        if (first == 0 && step == 0 && alike && width % 8 == 0 && others) return kEights;
        return alike && width >= kFewestShifted ? kShifted : kSingles;
    }
};
template <typename F>
void dispatch_run(int run, F&& f) {
    if (run == kEights) f(std::integral_constant<int, kEights>{});
    else if (run == kShifted) f(std::integral_constant<int, kShifted>{});
    else f(std::integral_constant<int, kSingles>{});
}
// Columns that the threads of a row have to reach over.
int reach(int width, int run) { return run == kShifted ? width + 7 : width; }
int threads_for(int cols, int groups) { return std::max(64, (ceil_div(cols, 8 * groups) + 31) / 32 * 32); }
template <int kThreads>
int blocks_for(int rows) { return in_lanes(kThreads) ? ceil_div(rows, kLaneThreads / kThreads) : rows; }

template <typename T, int kRun, bool kBlocks>
int quantize(const T* x, long long ldx, int rows, int cols, int8_t* codes, long long ldc, float* scales, cudaStream_t s) {
    const auto with = [&](auto threads, int block, auto groups) {
        constexpr int kThreads = decltype(threads)::value;
        launch_pdl(q8_quantize_kernel<T, kRun, kThreads, decltype(groups)::value, kBlocks>, dim3(blocks_for<kThreads>(rows)), dim3(block), 0, s, x, ldx, rows, cols, codes, ldc, scales);
    };
    const std::integral_constant<int, 0> any;
    const std::integral_constant<int, kQuantGroups> four;
    const int n = ceil_div(reach(cols, kRun), 8 * kQuantGroups);
    // The rows of one matrix lie alike, so that those one by one are the short ones: the lanes of a warp hold them.
    static_assert(32 * 8 * kQuantGroups >= kFewestShifted - 1);
    if (n > kBlockThreads) {
        launch_pdl(q8_quantize_loop_kernel<T, kBlocks>, dim3(rows), dim3(kLoopThreads), 0, s, x, ldx, cols, codes, ldc, scales);
    } else if constexpr (kRun == kShifted) {
        with(any, threads_for(reach(cols, kRun), kQuantGroups), four);
    } else if (n > 32) {
        // Up to 2048 values a warp holds too: 35484 x 1224 bf16 17.7 us, by blocks of two warps 37.2; 33213 x 2048 28.5 and 35.0;
        // fp32 32.3 and 38.1; 49.0 and 49.0.
        if constexpr (kRun == kSingles) B2_FAIL(B200ATTN_ERR_UNSUPPORTED, "q8_quantize: no kernel for %d columns one by one", cols);
        else if (n <= 64) with(std::integral_constant<int, 32>{}, kLaneThreads, std::integral_constant<int, 2 * kQuantGroups>{});
        else with(any, threads_for(cols, kQuantGroups), four);
    } else if (!kBlocks && n <= 4) {
        with(std::integral_constant<int, kBlocks ? 32 : 4>{}, kLaneThreads, four);
    } else if (!kBlocks && n <= 8) {
        with(std::integral_constant<int, kBlocks ? 32 : 8>{}, kLaneThreads, four);
    } else if (!kBlocks && n <= 16) {
        with(std::integral_constant<int, kBlocks ? 32 : 16>{}, kLaneThreads, four);
    } else {
        with(std::integral_constant<int, 32>{}, kLaneThreads, four);
    }
    B2_LAUNCH_CHECK();
    return 0;
}
template <bool kBlocks>
int quantize(ElemType t, const void* x, long long ldx, int rows, int cols, int8_t* codes, long long ldc, float* scales, cudaStream_t s) {
    if (rows == 0) return 0;
    int st = 0;
    dispatch_elem3(t, [&](auto tag) {
        using T = decltype(tag);
        Rows r;
        r.add(x, ldx, sizeof(T));
        dispatch_run(r.run(cols, reinterpret_cast<uintptr_t>(codes) % 8 == 0 && ldc % 8 == 0), [&](auto run) {
            st = quantize<T, decltype(run)::value, kBlocks>(static_cast<const T*>(x), ldx, rows, cols, codes, ldc, scales, s);
        });
    });
    return st;
}

template <typename X, typename T, int kRun>
int norm_block(const b200attn_norm_args& a, cudaStream_t s) {
    const auto with = [&](auto threads, auto groups, int block) {
        constexpr int kThreads = decltype(threads)::value;
        launch_pdl(norm_block_kernel<X, T, kRun, kThreads, decltype(groups)::value>, dim3(blocks_for<kThreads>(a.rows)), dim3(block), 0, s, a);
    };
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 2> two;
    const std::integral_constant<int, 4> four;
    const std::integral_constant<int, 0> any;
    const int reached = reach(a.width, kRun), n = ceil_div(reached, 8);
    if (n > 4 * kBlockThreads) {
        static PerDeviceOnce once;
        B2_PER_DEVICE_ONCE(once, B2_CUDA(cudaFuncSetAttribute(norm_block_loop_kernel<X, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormMostWidth * 4)));
        launch_pdl(norm_block_loop_kernel<X, T>, dim3(a.rows), dim3(kLoopThreads), (size_t)a.width * 4, s, a);
    } else if constexpr (kRun == kShifted) {
        if (n <= kBlockThreads) with(any, one, threads_for(reached, 1));
        else if (n <= 2 * kBlockThreads) with(any, two, threads_for(reached, 2));
        else with(any, four, threads_for(reached, 4));
    } else if (n <= 4) {
        with(std::integral_constant<int, 4>{}, one, kLaneThreads);
    } else if (n <= 8) {
        with(std::integral_constant<int, 8>{}, one, kLaneThreads);
    } else if (n <= 16) {
        with(std::integral_constant<int, 16>{}, one, kLaneThreads);
    } else if (n <= 32) {
        with(std::integral_constant<int, 32>{}, one, kLaneThreads);
    } else if constexpr (kRun == kEights) {
        // A thread per eight values as long as all rows are under way at once with them (64 registers each), else fewer threads that have more to wait for: 1000 x 4096
        // 10.3 us, with 512 threads a row 13.5.
        int sms = 0;
        B2_TRY(device_sm_count(&sms));
        const int few = sms * (1024 / threads_for(a.width, 1));
        if (n <= kBlockThreads && a.rows <= few) with(any, one, threads_for(a.width, 1));
        else if (n <= 64) with(std::integral_constant<int, 32>{}, two, kLaneThreads);
        else if (n <= 128) with(std::integral_constant<int, 32>{}, four, kLaneThreads);
        else if (n <= 2 * kBlockThreads) with(any, two, threads_for(a.width, 2));
        else with(any, four, threads_for(a.width, 4));
    } else {
        if (n <= 64) with(std::integral_constant<int, 64>{}, one, 64);
        else if (n <= 128) with(std::integral_constant<int, 128>{}, one, 128);
        else if (n <= kBlockThreads) with(std::integral_constant<int, kBlockThreads>{}, one, kBlockThreads);
        else if (n <= 2 * kBlockThreads) with(std::integral_constant<int, kBlockThreads>{}, two, kBlockThreads);
        else with(std::integral_constant<int, kBlockThreads>{}, four, kBlockThreads);
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
    Rows r;
    r.add(a.d_x, a.ldx, xb);
    if (a.d_x_out) r.add(a.d_x_out, a.ldx_out, xb);
    if (a.d_y) r.add(a.d_y, a.ldy, b);
    if (a.d_out) r.add(a.d_out, a.ld_out, b);
    if (a.d_gate && a.ld_gate) r.add(a.d_gate, a.ld_gate, b);
    bool others = a.d_gate && !a.ld_gate ? reinterpret_cast<uintptr_t>(a.d_gate) % 16 == 0 : true;
    for (const float* w : {a.d_post_w, a.d_pre_w}) others = others && reinterpret_cast<uintptr_t>(w) % 16 == 0;
    others = others && (!a.d_codes || (reinterpret_cast<uintptr_t>(a.d_codes) % 8 == 0 && a.ld_codes % 8 == 0));
    int st = 0;
    dispatch_elem3(type, [&](auto tag) {
        using T = decltype(tag);
        dispatch_run(r.run(a.width, others), [&](auto run) {
            constexpr int kRun = decltype(run)::value;
            st = x_type == ELEM_F32 ? norm_block<float, T, kRun>(a, s) : norm_block<T, T, kRun>(a, s);
        });
    });
    return st;
}

}  // namespace b200
