// Entry points of the 8-bit operators.
#include "gemm_pair.cuh"

#include <climits>
#include <new>

using namespace b200;

struct b200attn_q8_s {
    int out = 0, in = 0, act = -1, pitch = 0, scale_pitch = 0, device = 0;
    bool ready = false;
    int8_t* d_w = nullptr;       // in blocks (q8_block_offset), zeros behind column `in`; gated: up's rows from up_row() on
    float* d_scales = nullptr;   // [scale_pitch], gated: [2][scale_pitch]
    int* d_error = nullptr;
    int up_row() const { return (out + 7) / 8 * 8; }
    int rows() const { return act >= 0 ? 2 * up_row() : up_row(); }
};

namespace {

constexpr int kMostIn = 131072;              // 127 * 127 * in < 2^31
constexpr int kMostRows = INT_MAX - 1023;     // rounded up to whole tiles they are still ints
constexpr int kMostCols = INT_MAX - 1023;     // of the quantiser, whose threads walk a row by steps of up to 512: the first column behind it is still an int
constexpr int kPitchStep = 128;              // a slice of the products

bool elem_of(int dtype, ElemType* t) {
    *t = dtype == B200ATTN_DTYPE_F32 ? ELEM_F32 : dtype == B200ATTN_DTYPE_F16 ? ELEM_F16 : ELEM_BF16;
    return dtype == B200ATTN_DTYPE_BF16 || dtype == B200ATTN_DTYPE_F32 || dtype == B200ATTN_DTYPE_F16;
}
bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
int round_up(int v, int n) { return (v + n - 1) / n * n; }

// A handle is used on the device it was created on.
int check_handle(b200attn_q8 q, const char* what, bool need_weights) {
    B2_CHECK_ARG(q, "%s: null handle", what);
    int dev = 0;
    B2_CUDA(cudaGetDevice(&dev));
    B2_CHECK_ARG(dev == q->device, "%s: the handle belongs to device %d, device %d is current", what, q->device, dev);
    if (need_weights && !q->ready) B2_FAIL(B200ATTN_ERR_NOT_READY, "%s: weights not set", what);
    return 0;
}

// Codes and scales of rows that are quantised in front of the product.
size_t codes_bytes(b200attn_q8 q, int rows) { return ((size_t)rows * round_up(q->in, 16) + 255) / 256 * 256; }
size_t workspace_bytes(b200attn_q8 q, int rows, ElemType xt) {
    return rows == 0 || (q8_few_rows_takes(rows, q->in) && q8_few_rows_quantizes(rows, q->in, xt)) ? 0 : codes_bytes(q, rows) + (size_t)rows * 4;
}
int product(const Q8Product& p, cudaStream_t s) { return q8_few_rows_takes(p.rows, p.in) ? q8_few_rows(p, s) : gemm_pair_q8(s, p); }

Q8Product product_of(b200attn_q8 q, int rows, void* d_y, long long ldy, ElemType y_type, int accumulate) {
    Q8Product p;
    p.rows = rows; p.in = q->in; p.out = q->out; p.act = q->act;
    p.w = q->d_w; p.up_row = q->up_row(); p.w_rows = q->rows(); p.pitch = q->pitch; p.w_scales = q->d_scales; p.scale_pitch = q->scale_pitch;
    p.y = d_y; p.ldy = ldy; p.y_type = y_type; p.accumulate = accumulate != 0;
    p.error = q->d_error;
    return p;
}

int check_output(b200attn_q8 q, const char* what, int rows, const void* d_y, int y_dtype, long long ldy, int accumulate, ElemType* yt) {
    B2_CHECK_ARG(rows >= 0 && rows <= kMostRows, "%s: bad row count %d", what, rows);
    B2_CHECK_ARG(elem_of(y_dtype, yt), "%s: bad output type %d", what, y_dtype);
    B2_CHECK_ARG(rows == 0 || d_y, "%s: null output", what);
    B2_CHECK_ARG(ldy >= q->out, "%s: output pitch %lld below %d columns", what, ldy, q->out);
    B2_CHECK_ARG(aligned_to(d_y, elem_bytes(*yt)), "%s: output not aligned to its elements", what);
    B2_CHECK_ARG(!accumulate || (*yt == ELEM_F32 && q->act < 0), "%s: only plain products add to fp32 outputs", what);
    return 0;
}

}  // namespace

namespace b200 {
static bool q8_step(b200attn_q8 q, Q8Product p, const void* x, ElemType x_type, cudaStream_t s, int* status) {
    if (!q8_few_rows_takes(p.rows, q->in) || !q8_few_rows_quantizes(p.rows, q->in, x_type)) return false;
    p.x = x; p.ldx = q->in; p.x_type = x_type;
    p.late = false;
    *status = q8_few_rows(p, s);
    return true;
}
bool q8_step_norm(b200attn_q8 q, const float* x, const float* norm_w, float eps, int rows, __half* y, cudaStream_t s, int* status) {
    Q8Product p = product_of(q, rows, y, q->out, ELEM_F16, 0);
    p.norm_w = norm_w; p.eps = eps;
    return q8_step(q, p, x, ELEM_F32, s, status);
}
bool q8_step_residual(b200attn_q8 q, const __half* x, int rows, float* y, cudaStream_t s, int* status) {
    return q8_step(q, product_of(q, rows, y, q->out, ELEM_F32, 1), x, ELEM_F16, s, status);
}
}  // namespace b200

extern "C" int b200attn_q8_quantize(const void* d_x, int dtype, long long ldx, int rows, int cols, int8_t* d_codes, long long ld_codes, float* d_scales,
                                    b200attn_stream stream) {
    ElemType t;
    B2_CHECK_ARG(elem_of(dtype, &t), "q8_quantize: bad element type %d", dtype);
    B2_CHECK_ARG(rows >= 0 && rows <= kMostRows && cols > 0 && cols <= kMostCols, "q8_quantize: bad sizes %d x %d", rows, cols);
    B2_CHECK_ARG(ldx >= cols && ld_codes >= cols, "q8_quantize: pitch below %d columns", cols);
    if (rows == 0) return 0;
    B2_CHECK_ARG(d_x && d_codes && d_scales, "q8_quantize: null argument");
    B2_CHECK_ARG(aligned_to(d_x, elem_bytes(t)) && aligned_to(d_scales, 4), "q8_quantize: pointer not aligned to its elements");
    return launch_q8_quantize(t, d_x, ldx, rows, cols, d_codes, ld_codes, d_scales, as_stream(stream));
}

extern "C" int b200attn_q8_create(int out, int in, int act, b200attn_q8* handle) {
    B2_CHECK_ARG(handle, "q8_create: null argument");
    B2_CHECK_ARG(out > 0 && out <= INT_MAX / 2 - 512 && in > 0, "q8_create: bad sizes %d x %d", out, in);
    B2_CHECK_ARG(act < 0 || act == B200ATTN_ACT_GELU_TANH || act == B200ATTN_ACT_SILU, "q8_create: unknown activation %d", act);
    if (in > kMostIn) B2_FAIL(B200ATTN_ERR_UNSUPPORTED, "q8_create: depth %d above %d", in, kMostIn);
    refresh_runtime_flags();
    auto* q = new (std::nothrow) b200attn_q8_s();
    if (!q) B2_FAIL(B200ATTN_ERR_NOMEM, "q8_create: host allocation failed");
    q->out = out; q->in = in; q->act = act < 0 ? -1 : act;
    q->pitch = round_up(in, kPitchStep);
    q->scale_pitch = round_up(out, 256);                 // products read scales by whole tiles
    auto fill = [&]() -> int {
        B2_CUDA(cudaGetDevice(&q->device));
        B2_CUDA(cudaMalloc(&q->d_w, (size_t)q->rows() * q->pitch));
        B2_CUDA(cudaMalloc(&q->d_scales, (size_t)q->scale_pitch * (q->act >= 0 ? 8 : 4)));
        B2_CUDA(cudaMalloc(&q->d_error, 4));
        B2_CUDA(cudaMemset(q->d_error, 0, 4));
        B2_CUDA(cudaStreamSynchronize(cudaStreamLegacy));
        return 0;
    };
    const int st = fill();
    if (st != 0) { b200attn_q8_destroy(q); return st; }
    *handle = q;
    return 0;
}

extern "C" int b200attn_q8_destroy(b200attn_q8 q) {
    if (!q) return 0;
    cudaFree(q->d_w); cudaFree(q->d_scales); cudaFree(q->d_error);
    delete q;
    return 0;
}

extern "C" int b200attn_q8_set_weights(b200attn_q8 q, const void* d_w, const void* d_up, int dtype, long long ld, b200attn_stream stream) {
    ElemType t;
    B2_TRY(check_handle(q, "q8_set_weights", false));
    B2_CHECK_ARG(elem_of(dtype, &t), "q8_set_weights: bad element type %d", dtype);
    B2_CHECK_ARG(d_w && (q->act < 0) == (d_up == nullptr), "q8_set_weights: %s", q->act < 0 ? "one matrix wanted" : "gate and up matrices wanted");
    B2_CHECK_ARG(ld >= q->in, "q8_set_weights: pitch %lld below %d columns", ld, q->in);
    B2_CHECK_ARG(aligned_to(d_w, elem_bytes(t)) && aligned_to(d_up, elem_bytes(t)), "q8_set_weights: pointer not aligned to its elements");
    cudaStream_t s = as_stream(stream);
    q->ready = false;
    B2_TRY(launch_q8_quantize_weights(t, d_w, ld, q->out, q->in, q->d_w, q->pitch, q->d_scales, s));
    if (d_up)
        B2_TRY(launch_q8_quantize_weights(t, d_up, ld, q->out, q->in, q->d_w + (size_t)q->up_row() * q->pitch, q->pitch, q->d_scales + q->scale_pitch, s));
    B2_CUDA(cudaStreamSynchronize(s));
    q->ready = true;
    return 0;
}

extern "C" int b200attn_q8_export(b200attn_q8 q, int8_t* d_codes, float* d_scales, b200attn_stream stream) {
    B2_TRY(check_handle(q, "q8_export", true));
    B2_CHECK_ARG(d_codes && d_scales, "q8_export: null argument");
    B2_TRY(launch_q8_unblock(q->d_w, q->pitch, q->out, q->in, d_codes, as_stream(stream)));
    if (q->act >= 0)
        B2_TRY(launch_q8_unblock(q->d_w + (size_t)q->up_row() * q->pitch, q->pitch, q->out, q->in, d_codes + (size_t)q->out * q->in, as_stream(stream)));
    B2_CUDA(cudaMemcpy2DAsync(d_scales, (size_t)q->out * 4, q->d_scales, (size_t)q->scale_pitch * 4, (size_t)q->out * 4, q->act >= 0 ? 2 : 1, cudaMemcpyDeviceToDevice,
                              as_stream(stream)));
    return 0;
}

extern "C" int b200attn_q8_workspace(b200attn_q8 q, int rows, int x_dtype, size_t* bytes_out) {
    ElemType xt;
    B2_CHECK_ARG(q && bytes_out && rows >= 0 && rows <= kMostRows, "q8_workspace: bad argument");
    B2_CHECK_ARG(elem_of(x_dtype, &xt), "q8_workspace: bad input type %d", x_dtype);
    *bytes_out = workspace_bytes(q, rows, xt);
    return 0;
}

extern "C" int b200attn_q8_forward(b200attn_q8 q, const void* d_x, int x_dtype, long long ldx, int rows, void* d_y, int y_dtype, long long ldy, int accumulate,
                                   void* d_workspace, size_t workspace_size, b200attn_stream stream) {
    ElemType xt, yt;
    B2_TRY(check_handle(q, "q8_forward", true));
    B2_TRY(check_output(q, "q8_forward", rows, d_y, y_dtype, ldy, accumulate, &yt));
    B2_CHECK_ARG(elem_of(x_dtype, &xt), "q8_forward: bad input type %d", x_dtype);
    B2_CHECK_ARG(ldx >= q->in, "q8_forward: input pitch %lld below %d columns", ldx, q->in);
    if (rows == 0) return 0;
    B2_CHECK_ARG(d_x && aligned_to(d_x, elem_bytes(xt)), "q8_forward: input null or not aligned to its elements");
    Q8Product p = product_of(q, rows, d_y, ldy, yt, accumulate);
    cudaStream_t s = as_stream(stream);
    const size_t need = workspace_bytes(q, rows, xt);
    if (need == 0) {
        p.x = d_x; p.ldx = ldx; p.x_type = xt;
        return q8_few_rows(p, s);
    }
    B2_CHECK_ARG(d_workspace && aligned_to(d_workspace, 16) && workspace_size >= need, "q8_forward: a workspace of %zu bytes on a 16-byte boundary wanted", need);
    int8_t* codes = static_cast<int8_t*>(d_workspace);
    float* scales = reinterpret_cast<float*>(codes + codes_bytes(q, rows));
    p.codes = codes; p.ld_codes = round_up(q->in, 16); p.scales = scales;
    B2_TRY(launch_q8_quantize(xt, d_x, ldx, rows, q->in, codes, p.ld_codes, scales, s));
    return product(p, s);
}

extern "C" int b200attn_q8_forward_codes(b200attn_q8 q, const int8_t* d_codes, long long ld_codes, const float* d_scales, int rows, void* d_y, int y_dtype,
                                         long long ldy, int accumulate, b200attn_stream stream) {
    ElemType yt;
    B2_TRY(check_handle(q, "q8_forward_codes", true));
    B2_TRY(check_output(q, "q8_forward_codes", rows, d_y, y_dtype, ldy, accumulate, &yt));
    B2_CHECK_ARG(ld_codes >= q->in && ld_codes % 16 == 0, "q8_forward_codes: pitch %lld for %d columns, a multiple of 16 wanted", ld_codes, q->in);
    if (rows == 0) return 0;
    B2_CHECK_ARG(d_codes && d_scales, "q8_forward_codes: null argument");
    B2_CHECK_ARG(aligned_to(d_codes, 16) && aligned_to(d_scales, 4), "q8_forward_codes: codes not aligned to 16 bytes or scales to 4");
    Q8Product p = product_of(q, rows, d_y, ldy, yt, accumulate);
    p.codes = d_codes; p.ld_codes = ld_codes; p.scales = d_scales;
    return product(p, as_stream(stream));
}

extern "C" int b200attn_q8_device_status(b200attn_q8 q, int* code_out) {
    B2_TRY(check_handle(q, "q8_device_status", false));
    B2_CHECK_ARG(code_out, "q8_device_status: null argument");
    B2_CUDA(cudaDeviceSynchronize());
    B2_CUDA(cudaMemcpy(code_out, q->d_error, sizeof(int), cudaMemcpyDeviceToHost));
    if (*code_out != 0) B2_CUDA(cudaMemset(q->d_error, 0, sizeof(int)));
    return 0;
}

extern "C" int b200attn_norm_block(const b200attn_norm_args* args, b200attn_stream stream) {
    B2_CHECK_ARG(args, "norm_block: null argument");
    const b200attn_norm_args& a = *args;
    ElemType t, xt;
    B2_CHECK_ARG(elem_of(a.dtype, &t) && elem_of(a.x_dtype, &xt), "norm_block: bad element type");
    B2_CHECK_ARG(xt == t || xt == ELEM_F32, "norm_block: x is of the type of y or fp32");
    B2_CHECK_ARG(a.rows >= 0 && a.rows <= kMostRows && a.width > 0, "norm_block: bad sizes %d x %d", a.rows, a.width);
    if (a.width > kNormMostWidth) B2_FAIL(B200ATTN_ERR_UNSUPPORTED, "norm_block: width %d above %d", a.width, kNormMostWidth);
    B2_CHECK_ARG(a.ldx >= a.width && (!a.d_y || a.ldy >= a.width) && (!a.d_gate || a.ld_gate == 0 || a.ld_gate >= a.width) &&
                     (!a.d_x_out || a.ldx_out >= a.width) && (!a.d_out || a.ld_out >= a.width) && (!a.d_codes || a.ld_codes >= a.width),
                 "norm_block: a pitch is below the width %d", a.width);
    if (a.rows == 0) return 0;
    B2_CHECK_ARG(a.d_y || (!a.d_post_w && !a.d_gate), "norm_block: a norm or a gate of y without y");
    B2_CHECK_ARG(!a.d_gate || a.gate_kind == B200ATTN_GATE_AS_IS || a.gate_kind == B200ATTN_GATE_SIGMOID, "norm_block: unknown gate %d", a.gate_kind);
    B2_CHECK_ARG(a.d_x_out || a.d_out || a.d_codes, "norm_block: no output");
    B2_CHECK_ARG((a.d_codes != nullptr) == (a.d_scales != nullptr), "norm_block: codes and scales go together");
    B2_CHECK_ARG(a.d_x_out != a.d_x || a.ldx_out == a.ldx || !a.d_x, "norm_block: in place with another pitch");
    B2_CHECK_ARG(a.d_x, "norm_block: null x");
    B2_CHECK_ARG(aligned_to(a.d_x, elem_bytes(xt)) && aligned_to(a.d_x_out, elem_bytes(xt)) && aligned_to(a.d_y, elem_bytes(t)) && aligned_to(a.d_gate, elem_bytes(t)) &&
                     aligned_to(a.d_out, elem_bytes(t)) && aligned_to(a.d_post_w, 4) && aligned_to(a.d_pre_w, 4) && aligned_to(a.d_scales, 4),
                 "norm_block: a pointer is not aligned to its elements");
    return launch_norm_block(a, xt, t, as_stream(stream));
}
