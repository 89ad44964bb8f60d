// 8-bit operators: row quantiser and norm block (q8_rows.cu), products in 8-bit integers (q8_gemm.cu).
#pragma once

#include "elem.cuh"

namespace b200 {

// How a row of values v is held in 8 bits.  With a = max |v|: scale = a / 127, code = rint(v * (127 / a)), every operation rounded once to fp32, so that
// the codes do not depend on who computes them.  A row with a NaN or an infinity has the scale NaN and zero codes (what is made of it is NaN, not a
// plausible number); a row below 2^-116 the scale 0 and zero codes (127 / a would overflow).
struct Q8Row {
    float scale, inv;
};
constexpr uint32_t kQ8Finite = 0x7f800000u;              // bits of |v|: infinities and NaN from here on
constexpr float kQ8Tiny = 1.2037062152420224e-35f;       // 2^-116
__device__ __forceinline__ uint32_t q8_abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }      // ordered like |v|, NaN above all
__device__ __forceinline__ Q8Row q8_row(uint32_t abs_bits) {
    if (abs_bits >= kQ8Finite) return {__uint_as_float(0x7fc00000u), 0.f};
    const float a = __uint_as_float(abs_bits);
    if (a < kQ8Tiny) return {0.f, 0.f};
    return {__fdiv_rn(a, 127.0f), __fdiv_rn(127.0f, a)};
}
// inv = 0: a zero code, also of a NaN or an infinity (the conversion of a NaN is zero).
__device__ __forceinline__ int q8_code(float v, float inv) { return __float2int_rn(__fmul_rn(v, inv)); }
// Largest |value| of words of X: bits of fp32, or of two 16-bit values at a time, which are ordered like the values themselves; q8_max_bits makes bits of fp32 of it.
template <typename X>
__device__ __forceinline__ uint32_t q8_max_word(uint32_t top, uint32_t w) {
    return sizeof(X) == 4 ? max(top, w & 0x7fffffffu) : __vmaxu2(top, w & 0x7fff7fffu);
}
template <typename X>
__device__ __forceinline__ uint32_t q8_max_bits(uint32_t top) {
    if constexpr (sizeof(X) == 4) return top;
    const uint16_t bits = (uint16_t)max(top & 0xffffu, top >> 16);
    return q8_abs_bits(to_f32(*reinterpret_cast<const X*>(&bits)));
}

// Four codes in the bytes of a word.  1.5 * 2^23 added to a product of at most 127.00001 leaves its nearest integer, ties to even, in the low byte: the same as
// a conversion, at the rate of additions.
__device__ __forceinline__ uint32_t q8_codes4(float a, float b, float c, float d, float inv) {
    auto code = [&](float v) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.0f)); };
    const uint32_t ab = __byte_perm(code(a), code(b), 0x0040), cd = __byte_perm(code(c), code(d), 0x0040);
    return inv == 0.f ? 0u : __byte_perm(ab, cd, 0x5410);
}

// Codes of rows lie one behind the other (pitch ldc); those of weights in blocks of 8 rows x 128 columns, a block's rows of 128 bytes side by side and
// the blocks of eight rows one behind the other: what eight output columns want of K is one stretch of memory, and a block is the unit in which shared memory
// is swizzled for the tensor cores.
constexpr int kQ8Block = 8 * 128;
__host__ __device__ __forceinline__ size_t q8_block_offset(long long row, int col, int pitch) {
    return (size_t)(row / 8) * 8 * pitch + (size_t)(col / 128) * kQ8Block + row % 8 * 128 + col % 128;
}
int launch_q8_quantize(ElemType t, const void* x, long long ldx, int rows, int cols, int8_t* codes, long long ldc, float* scales, cudaStream_t s);
// pitch: columns rounded up to a multiple of 128, with zeros behind `cols`.
int launch_q8_quantize_weights(ElemType t, const void* w, long long ldw, int rows, int cols, int8_t* codes, int pitch, float* scales, cudaStream_t s);
int launch_q8_unblock(const int8_t* codes, int pitch, int rows, int cols, int8_t* out, cudaStream_t s);      // to rows of `cols`
constexpr int kNormMostWidth = 49152;                    // an fp32 row in shared memory
int launch_norm_block(const b200attn_norm_args& a, ElemType x_type, ElemType type, cudaStream_t s);

// Y = (X codes . W codes) * row scale * channel scale, or act(gate) * up of a pair of weights, from X itself (quantised on the way in).
struct Q8Product {
    const void* x = nullptr;         // [rows, in]
    long long ldx = 0;
    ElemType x_type = ELEM_F16;
    const float* norm_w = nullptr;   // fp32 X of up to 16 short rows (q8_few_rows_quantizes), fp16 Y: X is normalised first, with weights [in]
    float eps = 0.f;
    const int8_t* codes = nullptr;   // or X as codes, pitch a multiple of 16, and scales
    long long ld_codes = 0;
    const float* scales = nullptr;
    int rows = 0, in = 0, out = 0;
    const int8_t* w = nullptr;       // in blocks (q8_block_offset); gated: up's rows from `up_row` on, a multiple of 8
    int up_row = 0, w_rows = 0;      // w_rows: of all, a multiple of 8
    int pitch = 0;                   // a multiple of 128; columns behind `in` are zeros
    const float* w_scales = nullptr; // readable up to a whole tile of 256 (gated: of 128) columns
    int scale_pitch = 0;             // gated: from the gate's scales to those of up, a multiple of 4
    int act = -1;                    // b200attn_act of a gated pair, -1: plain
    void* y = nullptr;
    long long ldy = 0;
    ElemType y_type = ELEM_F32;
    bool accumulate = false;         // fp32 Y: added to what is there
    int* error = nullptr;
    bool late = true;                // few rows: the next launch is let in behind the wait (rows_enter)
};
bool q8_few_rows_takes(int rows, int in);      // the others: gemm_pair_q8, from codes
bool q8_few_rows_quantizes(int rows, int in, ElemType x_type);       // of those: X need not be codes
int q8_few_rows(const Q8Product& p, cudaStream_t s);
// The products of a decode step of few rows, a single launch each; false where they take more.  y = q of the normalised rows of x, fp16; y += q of fp16 x.
bool q8_step_norm(b200attn_q8 q, const float* x, const float* norm_w, float eps, int rows, __half* y, cudaStream_t s, int* status);
bool q8_step_residual(b200attn_q8 q, const __half* x, int rows, float* y, cudaStream_t s, int* status);

}  // namespace b200
