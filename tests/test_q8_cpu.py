"""CPU: the 8-bit operators refuse bad calls with the documented status before they touch a device."""
import ctypes as C

import pytest

P = C.c_void_p(4096)         # never dereferenced: every call below is refused, or has no rows


def refused(ops, status, text):
    assert status == ops.ERR_INVALID
    assert text in ops.lib().b200attn_last_error()


def test_quantize_refusals(ops):
    q = ops.lib().b200attn_q8_quantize
    ok = dict(x=4096, dtype=ops.DTYPE_BF16, ldx=64, rows=2, cols=64, codes=4096, ldc=64, scales=4096)

    def call(**kw):
        a = dict(ok, **kw)
        return q(a["x"], a["dtype"], a["ldx"], a["rows"], a["cols"], a["codes"], a["ldc"], a["scales"], None)
    for kw, text in ((dict(dtype=3), b"type"), (dict(dtype=-1), b"type"), (dict(rows=-1), b"sizes"), (dict(rows=2 ** 31 - 1), b"sizes"), (dict(cols=0), b"sizes"), (dict(ldx=63), b"pitch"),
                     (dict(ldc=63), b"pitch"), (dict(x=None), b"null"), (dict(codes=None), b"null"), (dict(scales=None), b"null"), (dict(x=4097), b"aligned"),
                     (dict(scales=4098), b"aligned"), (dict(dtype=ops.DTYPE_F32, x=4098), b"aligned")):
        refused(ops, call(**kw), text)
    assert call(rows=0) == 0 and call(rows=0, x=None, codes=None, scales=None) == 0


def test_product_refusals(ops):
    lib, h = ops.lib(), C.c_void_p()
    for out, inner, act in ((0, 64, -1), (64, 0, -1), (-1, 64, 0), (64, 64, 2), (2 ** 30, 64, -1)):
        refused(ops, lib.b200attn_q8_create(C.c_int(out), C.c_int(inner), C.c_int(act), C.byref(h)), b"q8_create")
    assert lib.b200attn_q8_create(C.c_int(8), C.c_int(131073), C.c_int(-1), C.byref(h)) == ops.ERR_UNSUPPORTED
    refused(ops, lib.b200attn_q8_create(C.c_int(8), C.c_int(8), C.c_int(-1), None), b"null")
    n = C.c_size_t()
    refused(ops, lib.b200attn_q8_workspace(None, 4, 0, C.byref(n)), b"q8_workspace")
    refused(ops, lib.b200attn_q8_forward(None, 4096, 0, 64, 2, 4096, 0, 64, 0, None, 0, None), b"null handle")
    refused(ops, lib.b200attn_q8_forward_codes(None, 4096, 64, 4096, 2, 4096, 0, 64, 0, None), b"null handle")
    refused(ops, lib.b200attn_q8_set_weights(None, 4096, None, 0, 64, None), b"null handle")
    refused(ops, lib.b200attn_q8_export(None, P, P, None), b"null handle")
    refused(ops, lib.b200attn_q8_device_status(None, None), b"null handle")
    assert lib.b200attn_q8_destroy(None) == 0


def norm_args(ops, **kw):
    a = ops.NormArgs(2, 64, ops.DTYPE_BF16, ops.DTYPE_F32, 4096, 64)
    a.d_y, a.ldy, a.x_scale, a.y_scale, a.eps = 8192, 64, 1.0, 1.0, 1e-6
    a.d_x_out, a.ldx_out, a.d_out, a.ld_out = 4096, 64, 16384, 64
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=5), b"type"), (dict(x_dtype=2), b"type of y or fp32"), (dict(rows=-1), b"sizes"), (dict(width=0), b"sizes"),
    (dict(ldx=63), b"pitch"), (dict(ldy=63), b"pitch"), (dict(ldx_out=10), b"pitch"), (dict(ld_out=63), b"pitch"), (dict(d_gate=4096, ld_gate=63), b"pitch"),
    (dict(d_y=None, d_post_w=4096), b"without y"), (dict(d_y=None, d_gate=4096), b"without y"), (dict(d_gate=4096, gate_kind=2), b"gate"),
    (dict(d_x_out=None, d_out=None), b"no output"), (dict(d_codes=4096, ld_codes=64), b"together"), (dict(d_scales=4096), b"together"),
    (dict(ldx_out=65), b"another pitch"), (dict(d_x=None), b"null x"), (dict(d_x=4098), b"aligned"), (dict(d_y=8193), b"aligned"), (dict(d_out=16385), b"aligned"),
    (dict(d_pre_w=4098), b"aligned"),
])
def test_norm_block_refusals(ops, kw, text):
    refused(ops, ops.lib().b200attn_norm_block(C.byref(norm_args(ops, **kw)), None), text)


def test_norm_block_limits(ops):
    lib = ops.lib()
    refused(ops, lib.b200attn_norm_block(None, None), b"null")
    a = norm_args(ops, width=49153, ldx=49153, ldy=49153, ldx_out=49153, ld_out=49153)
    assert lib.b200attn_norm_block(C.byref(a), None) == ops.ERR_UNSUPPORTED
    assert lib.b200attn_norm_block(C.byref(norm_args(ops, rows=0, d_x=None, d_x_out=4096)), None) == 0


def test_wrappers_want_tensors_of_the_device(ops):
    import torch
    x = torch.zeros(2, 64)
    for call in (lambda: ops.quantize_rows(x), lambda: ops.Int8Linear(x), lambda: ops.Int8GatedLinear(x, x), lambda: ops.norm_block(x, x, out_dtype=torch.float32),
                 lambda: ops.quantize_rows(x.double()), lambda: ops.Int8GatedLinear(x, x, 7)):
        with pytest.raises(ops.InvalidArgument):
            call()


@pytest.mark.parametrize("given,held", [(False, 0), (True, 1), (0, 0), (1, 1), (2, 2), (None, 0), (8, 1), ("yes", 1)])
def test_int8_weights_of_a_stack(ops, monkeypatch, given, held):
    """Whatever is true asks for 8-bit weights, as ever; 2 for 8-bit products too."""
    class Library:
        def __getattr__(self, name):
            return lambda *a: 0
    monkeypatch.setattr(ops, "_lib", Library())
    assert ops.HybridStack(1, 64, 64, 1, 16, 1, int8_weights=given).cfg.int8_weights == held
