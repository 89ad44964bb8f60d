// Products in 8-bit integers on mma.sync: Y = (X codes . W codes) * row scale * channel scale for up to 16 rows, which are quantised on the way in.
// The sums are 32-bit integers, so the order in which warps and lanes take K does not show.
#include "elem.cuh"
#include "ptx_utils.cuh"
#include "q8.cuh"

#include <algorithm>

namespace b200 {
namespace {

constexpr int kThreads = 512, kWarps = 16, kRows = 16;
constexpr int kMostK = 12800;                    // 16 rows of codes in shared memory

// d[16 x 8] += a[16 x 32] b[32 x 8]; which k a lane's bytes stand for does not matter as long as both operands agree.
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Rows 64 bytes apart modulo 128: the two rows that eight lanes read together fill the 32 banks.
__device__ __host__ __forceinline__ int codes_pitch(int pitch) { return pitch + 64; }

template <typename X, typename Y>
__global__ void __launch_bounds__(kThreads)
q8_few_rows_kernel(const Q8Product p) {
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int s_sum[2][kWarps][128];
    __shared__ float s_scale[kRows];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rows = p.rows, pitch = codes_pitch(p.pitch);
    int8_t* sx = reinterpret_cast<int8_t*>(smem);
    pdl_enter();
    {
        const int m = warp;                      // a warp per row
        int8_t* dst = sx + m * pitch;
        if (m >= rows) {
            for (int c = lane; c < p.pitch; c += 32) dst[c] = 0;
        } else if (p.codes) {
            const int8_t* src = p.codes + m * p.ld_codes;
            for (int c = lane; c < p.pitch; c += 32) dst[c] = c < p.in ? src[c] : 0;
            if (lane == 0) s_scale[m] = p.scales[m];
        } else {
            const X* src = static_cast<const X*>(p.x) + m * p.ldx;
            uint32_t top = 0;
            for (int c = lane; c < p.in; c += 32) top = max(top, q8_abs_bits(to_f32(src[c])));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const Q8Row q = q8_row(top);
            for (int c = lane; c < p.pitch; c += 32) dst[c] = c < p.in ? (int8_t)q8_code(to_f32(src[c]), q.inv) : 0;
            if (lane == 0) s_scale[m] = q.scale;
        }
    }
    __syncthreads();
    const int parts = p.act >= 0 ? 2 : 1;
    for (int tile = blockIdx.x; tile * 8 < p.out; tile += gridDim.x) {
        for (int part = 0; part < parts; ++part) {
            int acc[4] = {0, 0, 0, 0};
            const int n = tile * 8 + g;
            const int8_t* w = p.w + (long long)(part * p.out + min(n, p.out - 1)) * p.pitch;
            for (int k = 64 * warp; k < p.pitch; k += 64 * kWarps) {
                const uint4 b = *reinterpret_cast<const uint4*>(w + k + 16 * t);
                const uint4 a = *reinterpret_cast<const uint4*>(sx + g * pitch + k + 16 * t), a8 = *reinterpret_cast<const uint4*>(sx + (g + 8) * pitch + k + 16 * t);
                mma_s8(acc, a.x, a8.x, a.y, a8.y, b.x, b.y);
                mma_s8(acc, a.z, a8.z, a.w, a8.w, b.z, b.w);
            }
            int* out = s_sum[part][warp];
            out[g * 8 + 2 * t] = acc[0];
            out[g * 8 + 2 * t + 1] = acc[1];
            out[(g + 8) * 8 + 2 * t] = acc[2];
            out[(g + 8) * 8 + 2 * t + 1] = acc[3];
        }
        __syncthreads();
        if (threadIdx.x < 128) {
            const int m = threadIdx.x >> 3, n = tile * 8 + (threadIdx.x & 7);
            if (m < rows && n < p.out) {
                float v[2];
                for (int part = 0; part < parts; ++part) {
                    int sum = 0;
                    for (int i = 0; i < kWarps; ++i) sum += s_sum[part][i][threadIdx.x];
                    v[part] = (float)sum * s_scale[m] * p.w_scales[part * p.scale_pitch + n];
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
        __syncthreads();
    }
}

}  // namespace

bool q8_few_rows_takes(int rows, int in) { return rows <= kRows && in <= kMostK; }

int q8_few_rows(const Q8Product& p, cudaStream_t s) {
    int sms = 0, st = 0;
    B2_TRY(device_sm_count(&sms));
    dispatch_elem3(p.x_type, [&](auto xt) {
        dispatch_elem3(p.y_type, [&](auto yt) {
            using X = decltype(xt);
            using Y = decltype(yt);
            st = [&]() -> int {
                static PerDeviceOnce once;
                B2_PER_DEVICE_ONCE(once, B2_CUDA(cudaFuncSetAttribute(q8_few_rows_kernel<X, Y>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRows * (kMostK + 64))));
                const int tiles = ceil_div(p.out, 8);
                launch_pdl(q8_few_rows_kernel<X, Y>, dim3(std::min(tiles, sms)), dim3(kThreads), (size_t)kRows * codes_pitch(p.pitch), s, p);
                B2_LAUNCH_CHECK();
                return 0;
            }();
        });
    });
    return st;
}

}  // namespace b200
