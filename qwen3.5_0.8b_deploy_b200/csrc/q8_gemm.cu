// Products in 8-bit integers of up to 16 rows on mma.sync: Y = (X codes . W codes) * row scale * channel scale, X quantised on the way in.
//
// With so few rows a product is one pass over its weights, read straight into the registers of the lanes that multiply them: a warp takes tiles of eight
// output columns over a slice of K, a block of 8 x 128 codes in one access of 32 bytes a lane, several in flight while others are being multiplied.  The
// first ones are asked for before the wait on the preceding kernel (weights are complete when b200attn_q8_set_weights returns), so that they arrive while X is
// quantised.  Each CTA quantises all rows for itself: they are few, and a launch in front would cost more.
// The sums are 32-bit integers: slices of K meet in shared memory in any order with the same result.
//
// 1 x 1024 -> 2 x 3584 fp16 (7.3 MB) 3.5 us, 4.0 with the weights from memory; 16 x 4096 -> 4096 bf16 (16.8 MB) 7.4, of which quantising takes about 3: as a chain of
// one load, a maximum over the row and one store of codes it is the bound at 16 rows, at one row the chain from launch to the last sums.
#include "elem.cuh"
#include "ptx_utils.cuh"
#include "q8.cuh"

#include <algorithm>
#include <type_traits>

namespace b200 {
namespace {

constexpr int kThreads = 512, kWarps = 16, kRows = 16;
constexpr int kMostK = 8192;                     // 16 rows of codes in shared memory, and room for the next launch beside them
constexpr int kMostTiles = 64;                   // of a CTA
constexpr size_t kMostShared = (227 - 4) * 1024; // of a CTA, beside its static part

struct FewPlan {
    int units;                                   // eights of output columns
    int slices_log2;                             // slices of K; the warps of a slice share the tiles
};

// d[16 x 8] += a[16 x 32] b[32 x 8]; which k a lane's bytes stand for does not matter as long as both operands agree.
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
struct Weights { uint32_t v[8]; };
__device__ __forceinline__ void load_weights(const int8_t* p, Weights& w) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.u32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(w.v[0]), "=r"(w.v[1]), "=r"(w.v[2]), "=r"(w.v[3]), "=r"(w.v[4]), "=r"(w.v[5]), "=r"(w.v[6]), "=r"(w.v[7]) : "l"(p));
}

// Rows 16 bytes apart modulo 128: eight lanes read two rows, in each every other 16 bytes of 128.
__device__ __host__ __forceinline__ int codes_pitch(int pitch) { return pitch + 16; }
__device__ __forceinline__ int part_begin(int i, int n, int items) { return (int)((long long)i * items / n); }

// 16 bytes of a row from column k on, zeros behind it.
template <typename X>
__device__ __forceinline__ uint4 load_unit(const X* row, int k, int cols, bool aligned) {
    constexpr int kPer = 16 / (int)sizeof(X);
    if (aligned && k + kPer <= cols) return *reinterpret_cast<const uint4*>(row + k);
    __align__(16) X v[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = k + j < cols ? row[k + j] : from_f32<X>(0.f);
    return *reinterpret_cast<const uint4*>(v);
}
template <typename X>
__device__ __forceinline__ void unpack_unit(const uint4& u, float (&v)[16 / sizeof(X)]) {
    const X* p = reinterpret_cast<const X*>(&u);
#pragma unroll
    for (int j = 0; j < 16 / (int)sizeof(X); ++j) v[j] = to_f32(p[j]);
}

// Rows of X that lanes hold whole, as so many units each, while they look for the largest value.  Longer ones are quantised by a launch of their own: at 16
// rows of 8192 fp16 values a CTA would spend more time on them than on its weights (25.7 us against 13.9 for both launches; 16 x 4096 8.1 against 9.2).
constexpr int kUnits = 16, kUnitsShallow = 4;
__host__ __device__ __forceinline__ int row_share_log2(int rows) { return rows > 8 ? 0 : rows > 4 ? 1 : rows > 2 ? 2 : rows > 1 ? 3 : 4; }    // warps of a row
inline int units_wanted(int rows, int in, ElemType t) { return ceil_div(ceil_div(in * (int)elem_bytes(t), 512), 1 << row_share_log2(rows)); }

// All rows as codes into shared memory (zeros from column `in` on), their scales beside them.  kNorm: fp32 rows that are normalised first, as b200attn_norm_block
// makes codes of them: with the norm's weights (s_norm) multiplied in, and 1 / rms in the scale.
template <typename X, int kBatch, bool kNorm>
__device__ __forceinline__ void quantize_rows(const Q8Product& p, int8_t* sx, int pitch, float* s_scale, uint32_t* s_max, float* s_sum, const float* s_norm, int warp,
                                              int lane) {
    constexpr int kPer = 16 / (int)sizeof(X);
    const int share_log2 = row_share_log2(p.rows), share = 1 << share_log2;
    const int m = warp >> share_log2, sub = warp & (share - 1), step = 32 * kPer * share, first = kPer * (32 * sub + lane);
    const X* row = static_cast<const X*>(p.x) + (m < p.rows ? m : 0) * p.ldx;
    const bool aligned = reinterpret_cast<uintptr_t>(row) % 16 == 0;
    uint4 raw[kBatch];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) raw[i] = m < p.rows && first + i * step < p.in ? load_unit(row, first + i * step, p.in, aligned) : make_uint4(0, 0, 0, 0);
    float squares = 0.f;
    if constexpr (kNorm) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int k = first + i * step;
            if (k >= p.in) break;
            float4& x = reinterpret_cast<float4&>(raw[i]);
            const float4 w = *reinterpret_cast<const float4*>(s_norm + k);
            squares += (x.x * x.x + x.y * x.y) + (x.z * x.z + x.w * x.w);
            x = make_float4(__fmul_rn(x.x, w.x), __fmul_rn(x.y, w.y), __fmul_rn(x.z, w.z), __fmul_rn(x.w, w.w));
        }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
        for (const uint32_t w : {raw[i].x, raw[i].y, raw[i].z, raw[i].w}) top = q8_max_word<X>(top, w);
    top = q8_max_bits<X>(top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (kNorm) squares += __shfl_xor_sync(0xffffffffu, squares, o);
    }
    if (share > 1) {
        if (lane == 0) {
            s_max[warp] = top;
            s_sum[warp] = squares;
        }
        __syncthreads();
        squares = 0.f;
        for (int i = 0; i < share; ++i) {
            top = max(top, s_max[(m << share_log2) + i]);
            squares += s_sum[(m << share_log2) + i];
        }
    }
    const Q8Row q = q8_row(top);
    if (m < p.rows && sub == 0 && lane == 0) s_scale[m] = kNorm ? q.scale / sqrtf(squares / (float)p.in + p.eps) : q.scale;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
        const int k = first + i * step;
        if (k >= p.pitch) break;
        float v[kPer];
        unpack_unit<X>(raw[i], v);
        int8_t* dst = sx + m * pitch + k;
        if constexpr (kPer == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(q8_codes4(v[0], v[1], v[2], v[3], q.inv), q8_codes4(v[4], v[5], v[6], v[7], q.inv));
        else *reinterpret_cast<uint32_t*>(dst) = q8_codes4(v[0], v[1], v[2], v[3], q.inv);
    }
}

// kDeep: all registers of an SM for loads in flight, of weights and of long rows of X.  Otherwise half of them are left to the next launch.
template <typename X, typename Y, bool kDeep, bool kNorm>
__global__ void __launch_bounds__(kThreads, kDeep ? 1 : 2)
q8_few_rows_kernel(const Q8Product p, const FewPlan plan) {
    constexpr bool kCodes = std::is_same<X, int8_t>::value;                    // X comes as codes
    constexpr int kAhead = kDeep ? 4 : 2;                                      // blocks of 8 x 128 codes that a warp asks for at once
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ float s_scale[kRows], s_wscale[8 * kMostTiles];
    __shared__ uint32_t s_max[kWarps];
    __shared__ float s_sum[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int pitch = codes_pitch(p.pitch), parts = p.act >= 0 ? 2 : 1;
    int8_t* sx = reinterpret_cast<int8_t*>(smem);
    int* sums = reinterpret_cast<int*>(smem + kRows * pitch);                  // [slice][tile][4][32]: a lane's four sums of a tile
    const int u0 = part_begin(blockIdx.x, gridDim.x, plan.units), u1 = part_begin(blockIdx.x + 1, gridDim.x, plan.units);
    const int tiles = (u1 - u0) * parts;                                       // gated: the gate's and up's tile of a unit in turn
    const int slices = 1 << plan.slices_log2, slice = warp & (slices - 1), group = warp >> plan.slices_log2, groups = kWarps >> plan.slices_log2;
    const int chunks = p.pitch / 128, per = (chunks + slices - 1) / slices, c0 = min(chunks, slice * per), c1 = min(chunks, c0 + per);

    Weights ring[2][kAhead];
    int next_tile = group, next_c = c0;                                        // what is asked for next
    auto fetch = [&](auto& b) {
        if (next_tile >= tiles || c0 >= c1) return;
        const int unit = u0 + (parts == 2 ? next_tile >> 1 : next_tile), row = 8 * unit + (parts == 2 && next_tile & 1 ? p.up_row : 0);
        const int8_t* w = p.w + (long long)row * p.pitch + next_c * kQ8Block + 32 * lane;
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (next_c + i < c1) load_weights(w + i * kQ8Block, b[i]);
        next_c += kAhead;
        if (next_c >= c1) { next_c = c0; next_tile += groups; }
    };
    fetch(ring[0]);
    if constexpr (kCodes) fetch(ring[1]);                                      // X takes the registers otherwise
    for (int i = threadIdx.x; i < 8 * tiles; i += kThreads) {                  // the scales of this CTA's columns, [part][column]
        const int part = i >= 8 * (u1 - u0), n = 8 * u0 + i - part * 8 * (u1 - u0);
        s_wscale[i] = n < p.out ? p.w_scales[part * p.scale_pitch + n] : 0.f;
    }
    float* s_norm = reinterpret_cast<float*>(sums + ((size_t)tiles << plan.slices_log2) * 128);
    if constexpr (kNorm) {
        for (int i = threadIdx.x; i < p.in; i += kThreads) s_norm[i] = p.norm_w[i];
        __syncthreads();
    }
    rows_enter(p.late);
    if constexpr (kCodes) {
        for (int m = warp; m < kRows; m += kWarps) {
            const int8_t* src = p.codes + m * p.ld_codes;
            for (int k = 16 * lane; k < p.pitch; k += 512)
                *reinterpret_cast<uint4*>(sx + m * pitch + k) = m < p.rows && k < p.in ? *reinterpret_cast<const uint4*>(src + k) : make_uint4(0, 0, 0, 0);
            if (lane == 0 && m < p.rows) s_scale[m] = p.scales[m];
        }
    } else {
        quantize_rows<X, kDeep ? kUnits : kUnitsShallow, kNorm>(p, sx, pitch, s_scale, s_max, s_sum, s_norm, warp, lane);
    }
    __syncthreads();

    const bool high = p.rows > 8;
    const int8_t* xp = sx + g * pitch + 32 * t;
    int acc[4] = {0, 0, 0, 0}, tile = group, c = c0;
    auto multiply = [&](const auto& b) {
        if (tile >= tiles || c0 >= c1) return;
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (c + i < c1) {
                const uint4* x = reinterpret_cast<const uint4*>(xp + 128 * (c + i));
                const uint4* x8 = reinterpret_cast<const uint4*>(xp + 8 * pitch + 128 * (c + i));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 a = x[h];
                    uint4 a8 = make_uint4(0, 0, 0, 0);
                    if (high) a8 = x8[h];
                    mma_s8(acc, a.x, a8.x, a.y, a8.y, b[i].v[4 * h], b[i].v[4 * h + 1]);
                    mma_s8(acc, a.z, a8.z, a.w, a8.w, b[i].v[4 * h + 2], b[i].v[4 * h + 3]);
                }
            }
        c += kAhead;
        if (c < c1) return;
        int* out = sums + (slice * tiles + tile) * 128 + lane;
#pragma unroll
        for (int j = 0; j < 4; ++j) { out[32 * j] = acc[j]; acc[j] = 0; }
        c = c0;
        tile += groups;
    };
    while (tile < tiles && c0 < c1) {
        if constexpr (!kCodes) fetch(ring[1]);
        multiply(ring[0]);
        fetch(ring[0]);
        multiply(ring[1]);
        if constexpr (kCodes) fetch(ring[1]);
    }
    __syncthreads();
    const int used = min(slices, (chunks + per - 1) / per);                    // slices with chunks of their own
    for (int i = threadIdx.x; i < (u1 - u0) * 128; i += kThreads) {
        const int unit = i >> 7, at = i & 127, j = at >> 5, l = at & 31;
        const int m = (l >> 2) + 8 * (j >> 1), n = 8 * (u0 + unit) + 2 * (l & 3) + (j & 1);
        if (m >= p.rows || n >= p.out) continue;
        float v[2];
        for (int part = 0; part < parts; ++part) {
            int sum = 0;
            for (int s = 0; s < used; ++s) sum += sums[(s * tiles + unit * parts + part) * 128 + at];
            v[part] = (float)sum * s_scale[m] * s_wscale[8 * (part * (u1 - u0) + unit) + (n & 7)];
        }
        if (p.act == B200ATTN_ACT_SILU) v[0] = activated<float, B200ATTN_ACT_SILU>(v[0]) * v[1];
        if (p.act == B200ATTN_ACT_GELU_TANH) v[0] = activated<float, B200ATTN_ACT_GELU_TANH>(v[0]) * v[1];
        Y* y = static_cast<Y*>(p.y) + m * p.ldy + n;
        if constexpr (std::is_same<Y, float>::value) {
            if (p.accumulate) v[0] += *y;
        }
        *y = from_f32<Y>(v[0]);
    }
}

template <typename X, typename Y, bool kDeep, bool kNorm = false>
int launch_few_rows(const Q8Product& p, const FewPlan& plan, int grid, size_t smem, cudaStream_t s) {
    static PerDeviceOnce once;
    // The split of the L1 store that launch_pdl_split asks for with every launch, which takes the host 1 us each time.
    B2_PER_DEVICE_ONCE(once, B2_CUDA(cudaFuncSetAttribute(q8_few_rows_kernel<X, Y, kDeep, kNorm>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostShared));
                       B2_CUDA(cudaFuncSetAttribute(q8_few_rows_kernel<X, Y, kDeep, kNorm>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared)));
    launch_pdl(q8_few_rows_kernel<X, Y, kDeep, kNorm>, dim3(grid), dim3(kThreads), smem, s, p, plan);
    B2_LAUNCH_CHECK();
    return 0;
}

}  // namespace

bool q8_few_rows_takes(int rows, int in) { return rows <= kRows && in <= kMostK; }
bool q8_few_rows_quantizes(int rows, int in, ElemType t) { return units_wanted(rows, in, t) <= kUnits; }

int q8_few_rows(const Q8Product& p, cudaStream_t s) {
    int sms = 0, st = 0;
    B2_TRY(device_sm_count(&sms));
    const int parts = p.act >= 0 ? 2 : 1, chunks = p.pitch / 128;
    FewPlan plan;
    plan.units = ceil_div(p.out, 8);
    const int grid = std::max(std::min(plan.units, sms), ceil_div(plan.units * parts, kMostTiles));
    const int tiles = ceil_div(plan.units, grid) * parts;
    // The split of K with the fewest blocks on the busiest warp; of equal ones that with the fewest slices.  Not one whose sums a CTA does not hold: 17 tiles of 8192
    // columns in 16 slices would want 271 KB.  Unsplit, 64 tiles of 8192 columns take 197 KB with a norm's weights.
    const auto shared = [&](int slices_log2) { return (size_t)kRows * codes_pitch(p.pitch) + ((size_t)tiles << slices_log2) * 512 + (p.norm_w ? (size_t)p.in * 4 : 0); };
    long long busiest = 0;
    plan.slices_log2 = 0;
    for (int l = 0; l <= 4 && (l == 0 || shared(l) <= kMostShared); ++l) {
        const long long blocks = (long long)ceil_div(tiles, kWarps >> l) * ceil_div(chunks, 1 << l);
        if (l == 0 || blocks < busiest) { busiest = blocks; plan.slices_log2 = l; }
    }
    const size_t smem = shared(plan.slices_log2);
    if (smem > kMostShared) B2_FAIL(B200ATTN_ERR_UNSUPPORTED, "8-bit product: %zu bytes of shared memory for %d rows of %d columns", smem, p.rows, p.in);
    // More weights than the first fetches of a warp bring in several times over, or long rows of X.  4096 x 2 x 11008 at one row 18.3 us, shallow 21; 1024 x 2 x
    // 3584 at one row 5.4 us, shallow 4.2.
    const bool deep = busiest > 8 || (p.x && units_wanted(p.rows, p.in, p.x_type) > kUnitsShallow);
    auto launch = [&](auto xt) {
        dispatch_elem3(p.y_type, [&](auto yt) {
            using X = decltype(xt);
            using Y = decltype(yt);
            st = deep ? launch_few_rows<X, Y, true>(p, plan, grid, smem, s) : launch_few_rows<X, Y, false>(p, plan, grid, smem, s);
        });
    };
    if (p.norm_w) return deep ? launch_few_rows<float, __half, true, true>(p, plan, grid, smem, s) : launch_few_rows<float, __half, false, true>(p, plan, grid, smem, s);
    if (p.codes) launch(int8_t{});
    else dispatch_elem3(p.x_type, launch);
    return st;
}

}  // namespace b200
