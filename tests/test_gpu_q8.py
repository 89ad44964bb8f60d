"""GPU: the 8-bit operators against their definitions in 64 bits.

Codes are compared exactly: they are defined by 32-bit arithmetic of one operation at a time.  Sums of products of codes are integers, exact in
float64.  U = 2^-24 is half a step of fp32.
"""
import ctypes as C
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {torch.float32: U, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}     # steps of the subnormals
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rand(seed, *shape, std=1.0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).mul_(std)


def activations(seed, rows, cols, dtype, pitch=None, offset=0):
    """Rows of different size with a loud channel, as a window of a wider buffer filled with NaN."""
    x = rand(seed, rows, cols) * torch.exp(rand(seed + 1, rows, 1))
    x[:, cols // 3] *= 15.0
    if pitch is None:
        return x.to(dtype).cuda()
    buf = torch.full((rows * pitch + offset,), float("nan"), dtype=dtype, device="cuda")
    view = buf[offset:].view(rows, pitch)[:, :cols]
    view.copy_(x.to(dtype))
    return view


def define_codes(x):
    """Codes (float64 integers) and fp32 scales by definition, on the CPU."""
    x = x.detach().cpu().float()
    a = x.abs().amax(1)
    a = torch.where(torch.isnan(x).any(1), torch.full_like(a, float("nan")), a)
    bad, held = ~torch.isfinite(a), a >= 2.0 ** -116
    c127 = torch.tensor(127.0)
    inv = torch.where(held & ~bad, c127 / a, torch.zeros(1))
    scale = torch.where(bad, torch.full_like(a, float("nan")), torch.where(held, a / c127, torch.zeros(1)))
    codes = torch.round(torch.where(bad[:, None], torch.zeros(1), x) * inv[:, None])
    return codes.double(), scale


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=-7.0), torch.nan_to_num(b, nan=-7.0))


# ---- quantiser -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,pitch,offset", [(1, 1, None, 0), (3, 7, None, 0), (1, 3584, None, 0), (5, 31, 40, 3), (17, 1000, 1001, 1), (2, 16384, None, 0), (33, 1024, 1088, 8),
                                                    (4, 2056, 2057, 0), (300, 64, None, 0), (3, 40001, None, 0), (70000, 9, 10, 0)])
def test_quantize(ops, cuda, dtype, rows, cols, pitch, offset):
    x = activations(rows * cols, rows, cols, dtype, pitch, offset)
    codes, scales = ops.quantize_rows(x)
    want, s = define_codes(x)
    assert torch.equal(codes.cpu().double(), want) and torch.equal(scales.cpu(), s)
    assert codes.stride(0) % 16 == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [5, 1024, 9000])
def test_quantize_rows_out_of_the_ordinary(ops, cuda, dtype, cols):
    x = activations(3, 12, cols, dtype)
    x[0] = 0
    x[1, cols - 1] = float("inf")
    x[2, 0] = float("nan")
    x[3, cols // 2] = float("-inf")
    x[4], x[5] = float("nan"), float("inf")
    x[6] = torch.finfo(dtype).max
    x[7] = -torch.finfo(dtype).tiny                # fp16: held; the others lie below 2^-116
    x[8] = torch.finfo(dtype).smallest_normal * 0.5
    x[9] = 1.0
    x[10] = -3.0
    x[11, :] = 0
    x[11, 1] = torch.finfo(dtype).max
    codes, scales = ops.quantize_rows(x)
    want, s = define_codes(x)
    assert torch.equal(codes.cpu().double(), want) and same(scales.cpu(), s)
    assert torch.isnan(scales[[1, 2, 3, 4, 5]]).all() and (codes[1:6] == 0).all() and scales[0] == 0


def test_quantize_rounds_ties_to_even(ops, cuda):
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, 0.49999997]], device="cuda")
    codes, scales = ops.quantize_rows(x)
    assert codes.tolist() == [[127, 0, 2, 2, 0, -2, -2, 126, 0]] and scales.item() == 1.0


def test_quantize_leaves_what_lies_around_it(ops, cuda):
    x = activations(1, 5, 100, torch.bfloat16)
    codes = torch.full((7, 130), 77, dtype=torch.int8, device="cuda")
    scales = torch.full((7,), 77.0, device="cuda")
    assert ops.lib().b200attn_q8_quantize(x.data_ptr(), ops.DTYPE_BF16, 100, 5, 100, codes[1:].data_ptr(), 130, scales[1:].data_ptr(), ops._current_stream()) == 0
    want, s = define_codes(x)
    assert torch.equal(codes[1:6, :100].cpu().double(), want) and torch.equal(scales[1:6].cpu(), s)
    assert (codes[0] == 77).all() and (codes[6] == 77).all() and (codes[1:6, 100:] == 77).all() and scales[0] == 77 and scales[6] == 77


# ---- product --------------------------------------------------------------------------------------------------------------------
def product(codes, scale, w_codes, w_scale):
    """Exact sums times the scales, in float64 on the GPU."""
    return (codes.cuda() @ w_codes.cuda().T) * scale.double().cuda()[:, None] * w_scale.double().cuda()[None]


def within(got, want, bound, dtype):
    """bound: what the steps in 32 bits may be off by; the rounding to dtype comes on top."""
    limit = bound + HALF_STEP[dtype] * (want.abs() + bound) + SMALLEST[dtype]
    err = (got.double() - want).abs()
    bad = ~(err <= limit)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, worst {(err / limit).max():.3f} of the limit, first at {bad.nonzero()[0].tolist()}"


# (sum as fp32) * row scale * channel scale: three roundings, and the scale itself one each.  fp32 results are rounded by the last of them.
PLAIN = 5.1 * U


def glu_reference(g, u, act):
    """GELU as z s(2 sqrt(2/pi) (z + 0.044715 z^3)): 1 + tanh cancels for negative z, in float64 too."""
    return g * torch.sigmoid(g if act == 1 else (8 / math.pi) ** 0.5 * (g + 0.044715 * g ** 3)) * u


def glu_bound(g, u, act, dtype):
    """The activation f(z) = z s(p(z)) with s the sigmoid and p(z) = z (SiLU) or 2 sqrt(2/pi) (z + 0.044715 z^3).  An error of d in z's last places moves f by
    d (1 + |z p'(z)|) of itself, an error e of the exponential by e; |z p'| <= 3 |p|.  z: PLAIN; p has up to six roundings more; the exponential of the library is off by
    2^-22 and by the rounding of its argument, |p| U.  16-bit results may use the fast exponential (its argument in base 2 is rounded: 2 |p| U more, 2^-21) and divide
    (2^-22).  The products round four times."""
    z = g.abs()
    p = z if act == 1 else 1.6 * (z + 0.044715 * z ** 3)
    e = (3 * p + 1) * PLAIN + 7 * p * U + 2.0 ** -22 + (0 if dtype == torch.float32 else 2 * p * U + 2.0 ** -21 + 2.0 ** -22)
    f = glu_reference(g, torch.ones_like(u), act).abs()
    # where 1 + e^-p overflows or its quotient is subnormal, the result is (next to) zero in 32 bits
    return (f * (e + PLAIN + 4 * U) + z * 2.0 ** -125) * u.abs() * (1 + PLAIN)


SIZES = [(1, 64, 8), (1, 1, 1), (2, 17, 3), (1, 1024, 3584), (3, 1000, 2313), (16, 4096, 515), (15, 128, 64), (16, 7, 40), (17, 256, 96), (31, 1024, 129), (33, 130, 1000),
         (64, 2048, 256), (100, 999, 257), (128, 1024, 1024), (129, 72, 33), (255, 512, 640), (257, 384, 2000), (300, 8192, 31), (777, 1003, 511), (1025, 640, 300), (4, 12000, 90),
         (2000, 100, 1), (513, 33, 7), (7, 6000, 1000), (40, 20000, 50), (11, 20000, 50), (2, 131072, 9), (18, 131072, 9), (16, 8192, 100), (9, 4096, 70), (16, 2048, 30), (8, 8192, 60), (4, 8191, 50), (1, 8192, 4100), (2, 40, 100003), (20, 40, 50001)]


@pytest.mark.parametrize("rows,cols,out", SIZES)
@pytest.mark.parametrize("x_type,y_type", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float32), (torch.float32, torch.float32), (torch.float16, torch.float16),
                                           (torch.float32, torch.bfloat16)])
def test_linear(ops, cuda, rows, cols, out, x_type, y_type):
    w = rand(5, out, cols, std=0.02).bfloat16().cuda()
    x = activations(7, rows, cols, x_type, cols + 5, 3)
    layer = ops.Int8Linear(w)
    wc, ws = define_codes(w)
    got_c, got_s = layer.weight_codes()
    assert torch.equal(got_c.cpu().double(), wc) and torch.equal(got_s.cpu(), ws)
    xc, xs = define_codes(x)
    want = product(xc, xs, wc, ws)
    y = layer.forward(x, out_dtype=y_type)
    assert layer.device_status() == 0
    within(y, want, PLAIN * want.abs(), y_type)
    codes, scales = ops.quantize_rows(x)
    again = layer.forward_codes(codes, scales, out_dtype=y_type)
    assert torch.equal(again, y)
    assert torch.equal(layer.forward(x, out_dtype=y_type), y)
    assert layer.device_status() == 0


@pytest.mark.parametrize("rows,cols,out", SIZES)
@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("y_type", TYPES)
def test_gated(ops, cuda, rows, cols, out, act, y_type):
    gate, up = (rand(s, out, cols, std=1.2 * cols ** -0.5).bfloat16().cuda() for s in (5, 6))
    x = activations(7, rows, cols, torch.bfloat16)
    layer = ops.Int8GatedLinear(gate, up, act)
    xc, xs = define_codes(x)
    g, u = (product(xc, xs, *define_codes(w)) for w in (gate, up))
    y = layer.forward(x, out_dtype=y_type)
    assert layer.device_status() == 0
    within(y, glu_reference(g, u, act), glu_bound(g, u, act, y_type), y_type)
    assert torch.equal(layer.forward_codes(*ops.quantize_rows(x), out_dtype=y_type), y)


@pytest.mark.parametrize("rows,cols,out,gated", [(1, 8192, 14232, False), (16, 6144, 18992, False), (3, 2048, 28456, False), (1, 8192, 14232, True), (16, 1024, 30808, True)])
def test_few_rows_whose_sums_fill_shared_memory(ops, cuda, rows, cols, out, gated):
    """One output column tile more than a whole number of warps has, on long rows: the split of K that keeps all warps busy has more sums than a CTA holds."""
    ws = [rand(s, out, cols, std=1.2 * cols ** -0.5).bfloat16().cuda() for s in (5, 6)[:1 + gated]]
    x = activations(7, rows, cols, torch.float16)
    xc, xs = define_codes(x)
    sums = [product(xc, xs, *define_codes(w)) for w in ws]
    if gated:
        y = ops.Int8GatedLinear(*ws, 1).forward(x, out_dtype=torch.float32)
        within(y, glu_reference(*sums, 1), glu_bound(*sums, 1, torch.float32), torch.float32)
    else:
        y = ops.Int8Linear(ws[0]).forward(x, out_dtype=torch.float32)
        within(y, sums[0], PLAIN * sums[0].abs(), torch.float32)


@pytest.mark.parametrize("rows", [1, 16, 40, 300])
@pytest.mark.parametrize("out,pitch", [(1024, 1024), (33, 37), (256, 260)])
def test_accumulate(ops, cuda, rows, out, pitch):
    w, x = rand(5, out, 512, std=0.02).cuda(), activations(7, rows, 512, torch.float16)
    layer = ops.Int8Linear(w)
    before = rand(9, rows, pitch).cuda()
    y = before.clone()
    layer.forward(x, out=y[:, :out], accumulate=True)
    want = product(*define_codes(x), *define_codes(w))
    total = want + before[:, :out].double()
    within(y[:, :out], total, PLAIN * want.abs(), torch.float32)
    assert torch.equal(y[:, out:], before[:, out:])


@pytest.mark.parametrize("rows,out", [(1, 40), (16, 515), (50, 100), (128, 64), (300, 515), (300, 512), (700, 1)])
@pytest.mark.parametrize("act", [-1, 1])
@pytest.mark.parametrize("y_type", TYPES)
@pytest.mark.parametrize("pad", [0, 1, 16])
def test_product_leaves_what_lies_around_it(ops, cuda, rows, out, act, y_type, pad):
    ws = [rand(s, out, 200, std=0.05).cuda() for s in (5, 6)]
    layer = ops.Int8Linear(ws[0]) if act < 0 else ops.Int8GatedLinear(*ws, act)
    x = activations(7, rows, 200, torch.bfloat16)
    y = torch.full((rows + 2, out + pad), 77.0, dtype=y_type, device="cuda")
    layer.forward(x, out=y[1:rows + 1, :out])
    assert torch.equal(y[1:rows + 1, :out].contiguous(), layer.forward(x, out_dtype=y_type))
    assert (y[0] == 77).all() and (y[rows + 1] == 77).all() and (y[1:rows + 1, out:] == 77).all()


@pytest.mark.parametrize("rows", [3, 16, 60, 400])
def test_rows_without_a_value(ops, cuda, rows):
    """Zero rows give zeros, rows with a NaN or an infinity NaN, and neither touches its neighbours."""
    w = rand(5, 96, 256).cuda()
    layer = ops.Int8Linear(w)
    x = activations(7, rows, 256, torch.bfloat16)
    clean = layer.forward(x)
    x[0] = 0
    x[2, 100] = float("inf")
    y = layer.forward(x)
    assert (y[0] == 0).all() and torch.isnan(y[2]).all()
    keep = [i for i in range(rows) if i not in (0, 2)]
    assert torch.equal(y[keep], clean[keep])
    w[7] = 0
    w[9, 3] = float("nan")
    y = ops.Int8Linear(w).forward(x)
    assert (y[1, 7] == 0) and torch.isnan(y[1, 9]) and torch.isfinite(y[1, [6, 8, 10]]).all()


def test_largest_sums(ops, cuda):
    """127 * 127 * 131072 = 2114060288 is the largest sum there is."""
    w = torch.ones(9, 131072, device="cuda")
    for rows in (1, 20):
        x = torch.ones(rows, 131072, device="cuda")
        x[0] = -1
        want = torch.full((rows, 9), 131072.0, dtype=torch.float64, device="cuda")
        want[0] *= -1
        within(ops.Int8Linear(w).forward(x), want, PLAIN * want.abs(), torch.float32)


def test_no_rows(ops, cuda):
    layer = ops.Int8Linear(rand(5, 40, 64).cuda())
    x = torch.empty(0, 64, device="cuda")
    assert layer.forward(x).shape == (0, 40)
    codes, scales = ops.quantize_rows(x)
    assert codes.shape == (0, 64) and scales.shape == (0,)
    assert layer.forward_codes(codes, scales).shape == (0, 40)
    assert [t.shape[0] for t in ops.norm_block(x, x, out_dtype=torch.float32)] == [0, 0]


def test_refusals_on_the_device(ops, cuda):
    layer = ops.Int8Linear(rand(5, 40, 64).cuda())
    gated = ops.Int8GatedLinear(rand(5, 40, 64).cuda(), rand(6, 40, 64).cuda())
    x = torch.zeros(20, 64, device="cuda")
    calls = [lambda: layer.forward(x[:, :63]), lambda: layer.forward(x.t()), lambda: layer.forward(x, out_dtype=torch.float64), lambda: layer.forward(x.cpu()),
             lambda: layer.forward(x, out=torch.zeros(20, 41, device="cuda")), lambda: layer.forward(x, accumulate=True),
             lambda: layer.forward(x, out=torch.zeros(20, 40, device="cuda", dtype=torch.float16), accumulate=True),
             lambda: gated.forward(x, out=torch.zeros(20, 40, device="cuda"), accumulate=True), lambda: layer.forward(x[:1].expand(20, 64)),
             lambda: layer.forward_codes(x, x[:, 0].contiguous()), lambda: layer.forward_codes(torch.zeros(20, 64, dtype=torch.int8, device="cuda"), x[:, 0]),
             lambda: layer.forward_codes(torch.zeros(20, 66, dtype=torch.int8, device="cuda")[:, :64], torch.zeros(20, device="cuda")),
             lambda: layer.forward_codes(torch.zeros(20 * 64 + 1, dtype=torch.int8, device="cuda")[1:].view(20, 64), torch.zeros(20, device="cuda")),
             lambda: ops.Int8GatedLinear(x, x[:19]), lambda: ops.Int8GatedLinear(x, x.half()), lambda: ops.norm_block(x, x[:19], out_dtype=torch.float32),
             lambda: ops.norm_block(x, x, out_dtype=torch.float16), lambda: ops.norm_block(x, x.half(), gate=x, out_dtype=torch.float16),
             lambda: ops.norm_block(x, x, pre_w=x[0, :63], out_dtype=torch.float32), lambda: ops.norm_block(x, gate=x, out_dtype=torch.float32),
             lambda: ops.norm_block(x.half(), x.bfloat16(), out_dtype=torch.bfloat16)]
    for i, call in enumerate(calls):
        with pytest.raises(ops.InvalidArgument):
            call()
            pytest.fail(f"call {i} was taken")
    n = C.c_size_t()
    assert ops.lib().b200attn_q8_workspace(layer.h, 20, ops.DTYPE_F32, C.byref(n)) == 0
    if n.value:
        y = torch.zeros(20, 40, device="cuda")
        ws = torch.empty(n.value + 16, dtype=torch.uint8, device="cuda")
        for p, size in ((None, n.value), (ws.data_ptr(), n.value - 1), (ws.data_ptr() + 8, n.value)):
            assert ops.lib().b200attn_q8_forward(layer.h, x.data_ptr(), ops.DTYPE_F32, 64, 20, y.data_ptr(), ops.DTYPE_F32, 40, 0, p, size, None) == ops.ERR_INVALID
    h = C.c_void_p()
    assert ops.lib().b200attn_q8_create(C.c_int(40), C.c_int(64), C.c_int(-1), C.byref(h)) == 0
    assert ops.lib().b200attn_q8_forward(h, x.data_ptr(), ops.DTYPE_F32, 64, 1, x.data_ptr(), ops.DTYPE_F32, 64, 0, None, 0, None) == ops.ERR_NOT_READY
    assert ops.lib().b200attn_q8_destroy(h) == 0


# ---- norm block -------------------------------------------------------------------------------------------------------------------
def norm_reference(x, y, pre, post, gate, sigmoid, xs, ys, eps):
    """float64 on the GPU: x', n, and bounds for both (without the final rounding)."""
    width = x.shape[1]
    # A root mean square in fp32: each square and the mean are rounded, and a thread adds at most 192 squares before the sums of 256 threads meet in
    # 13 steps, so that the mean is off by less than (192 + 13 + 3) U of itself and its root by half of that; root, quotient and eps add 4.
    rms_err = (min(width, 192) + 16) / 2 * U + 4 * U
    ax = (xs * x.double()).abs()
    if y is None:
        z, ez = torch.zeros_like(ax), torch.zeros_like(ax)
    else:
        z = y.double()
        ez = torch.zeros_like(z)
        if post is not None:
            z = z / torch.sqrt(z.square().mean(1, keepdim=True) + eps) * post.double()
            ez = z.abs() * (rms_err + 3 * U)
        if gate is not None:
            g = gate.double()
            # sigmoid: the exponential is off by 2^-22, sum and quotient round
            ez = ez * (torch.sigmoid(g) if sigmoid else g.abs()) + z.abs() * (torch.sigmoid(g) * (2.0 ** -22 + 3 * U) + 2.0 ** -125 if sigmoid else g.abs() * U)
            z = z * (torch.sigmoid(g) if sigmoid else g)
    new = float(torch.tensor(xs)) * x.double() + float(torch.tensor(ys)) * z
    e_new = ax * U + abs(ys) * (ez + z.abs() * 2 * U) + new.abs() * U
    inv = 1 / torch.sqrt(new.square().mean(1, keepdim=True) + eps)
    n = new * inv * (1 if pre is None else pre.double())
    # errors of x' move the root mean square by at most their own root mean square
    e_rms = e_new.square().mean(1, keepdim=True).sqrt() * inv
    e_n = (e_new * inv) * (1 if pre is None else pre.double().abs()) + n.abs() * (e_rms + rms_err + 3 * U)
    return new, e_new * 1.01, n, e_n * 1.01, inv, e_rms + rms_err


def norm_inputs(rows, width, dtype, x_type, post, gate, pitch=0):
    x = activations(11, rows, width, x_type, width + pitch if pitch else None)
    y = activations(13, rows, width, dtype, width + pitch if pitch else None)
    if rows > 3:
        y[2], x[3] = 0, 0
    pre = (1 + rand(17, width, std=0.1)).cuda()
    post = (1 + rand(19, width, std=0.1)).cuda() if post else None
    g = None if not gate else rand(23, *((width,) if gate == "channel" else (rows, width)), std=2.0).to(dtype).cuda()
    return x, y, pre, post, g


NORM_SIZES = [(1, 1), (1, 1024), (4, 7), (3, 130), (5, 1023), (2, 2050), (9, 4096), (7, 5000), (2, 8192), (3, 8200), (2, 20001), (300, 256), (1, 49152), (66000, 12), (1024, 1024), (1025, 1024), (1100, 520), (1030, 1001), (1500, 4096), (1200, 2050),
              (1100, 10000)]


@pytest.mark.parametrize("rows,width", NORM_SIZES)
@pytest.mark.parametrize("dtype,x_type", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                          (torch.float16, torch.float32)])
@pytest.mark.parametrize("post,gate,xs,ys", [(False, "", 1.0, 1.0), (True, "", 1.0, 1.0), (True, "sigmoid", 1.0, 0.25), (False, "channel", 0.9, 1.5), (True, "token", 0.5, -1.0)])
def test_norm_block(ops, cuda, rows, width, dtype, x_type, post, gate, xs, ys):
    x, y, pre, post, g = norm_inputs(rows, width, dtype, x_type, post, gate, pitch=width % 3)
    eps = 1e-6
    new, e_new, n, e_n, _, _ = norm_reference(x, y, pre, post, g, gate == "sigmoid", xs, ys, eps)
    got_x, got_n = ops.norm_block(x, y, pre, post, g, gate == "sigmoid", xs, ys, eps, out_dtype=dtype)
    within(got_x, new, e_new, x_type)
    within(got_n, n, e_n, dtype)
    kept = x.clone()
    again_x, again_n = ops.norm_block(kept, y, pre, post, g, gate == "sigmoid", xs, ys, eps, out_dtype=dtype, in_place=True)
    assert again_x is kept and torch.equal(kept, got_x) and torch.equal(again_n, got_n)


@pytest.mark.parametrize("rows,width", NORM_SIZES)
@pytest.mark.parametrize("dtype,x_type", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("gate,xs,ys", [("", 1.0, 1.0), ("channel", 0.9, 1.5), ("token", 1.0, -0.3)])
def test_norm_block_codes(ops, cuda, rows, width, dtype, x_type, gate, xs, ys):
    """Without a norm behind the block every step in front of the codes is one rounding per element, so that they are known exactly."""
    x, y, pre, _, g = norm_inputs(rows, width, dtype, x_type, False, gate, pitch=width % 2)
    got_x, codes, scales = ops.norm_block(x, y, pre, None, g, False, xs, ys)
    z = y.cpu().float()
    if g is not None:
        z = z * g.cpu().float()
    new = x.cpu().float() * torch.tensor(xs) + z * torch.tensor(ys)
    assert torch.equal(got_x.cpu(), new.to(x_type))
    want, s = define_codes(new * pre.cpu())
    assert torch.equal(codes.cpu().double(), want)
    _, _, _, _, inv, e_inv = norm_reference(x, y, pre, None, g, False, xs, ys, 1e-6)
    ideal = s.double().cuda() * inv[:, 0]
    within(scales, ideal, ideal.abs() * (e_inv[:, 0] + 3 * U), torch.float32)


@pytest.mark.parametrize("width", [64, 1000, 3000])
def test_norm_block_parts(ops, cuda, width):
    """No block output, no weights, only the update, only the norm; the codes of a sandwich agree with its typed result."""
    x, y, pre, post, _ = norm_inputs(6, width, torch.float32, torch.float32, True, "")
    new, e_new, n, e_n, _, _ = norm_reference(x, None, pre, None, None, False, 1.0, 1.0, 1e-5)
    got_x, got_n = ops.norm_block(x, pre_w=pre, eps=1e-5, out_dtype=torch.float32)
    assert torch.equal(got_x, x)
    within(got_n, n, e_n, torch.float32)
    _, _, n, e_n, _, _ = norm_reference(x, y, None, None, None, False, 1.0, 1.0, 1e-6)
    within(ops.norm_block(x, y, out_dtype=torch.float32)[1], n, e_n, torch.float32)
    a = ops.NormArgs(6, width, ops.DTYPE_F32, ops.DTYPE_F32, x.data_ptr(), width)
    a.d_y, a.ldy, a.x_scale, a.y_scale, a.eps = y.data_ptr(), width, 1.0, 1.0, 1e-6
    keep = torch.full((8, width + 3), 77.0, device="cuda")
    a.d_x_out, a.ldx_out = keep[1:].data_ptr(), width + 3
    assert ops.lib().b200attn_norm_block(C.byref(a), ops._current_stream()) == 0
    assert torch.equal(keep[1:7, :width], x + y) and (keep[0] == 77).all() and (keep[7] == 77).all() and (keep[1:7, width:] == 77).all()
    typed = ops.norm_block(x, y, pre, post, out_dtype=torch.float32)[1]
    _, codes, scales = ops.norm_block(x, y, pre, post)
    # a code is off by half a step and what 32 bits lose
    assert ((codes.float() * scales[:, None] - typed).abs() <= 0.51 * scales[:, None] + 1e-30).all()


PLACES = [(0, 0), (1, 0), (3, 5), (0, 1), (8, 8)]      # values in front of the first row, and behind each
WIDTHS = [1, 2, 5, 8, 9, 16, 31, 33, 64, 100, 129, 249, 250, 256, 257, 263, 511, 520, 1017, 1024, 1027, 2041, 4089, 4090, 4097, 8185, 8190, 16377, 16380]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset,pad", PLACES)
def test_quantize_wherever_rows_lie(ops, cuda, dtype, offset, pad):
    for rows in (1, 3, 37):
        for cols in WIDTHS:
            x = activations(rows + cols, rows, cols, dtype, cols + pad, offset)
            want, s = define_codes(x)
            for pitch, at in ((cols, 0), (cols + 3, 1), ((cols + 15) // 16 * 16, 0)):
                codes = torch.full((rows * pitch + at + 16,), 77, dtype=torch.int8, device="cuda")
                scales = torch.full((rows + 1,), 77.0, device="cuda")
                assert ops.lib().b200attn_q8_quantize(x.data_ptr(), ops._Q8_DTYPES[dtype], cols + pad, rows, cols, codes[at:].data_ptr(), pitch, scales.data_ptr(),
                                                      ops._current_stream()) == 0
                got = codes[at:at + rows * pitch].view(rows, pitch)
                assert torch.equal(got[:, :cols].cpu().double(), want) and torch.equal(scales[:rows].cpu(), s), (rows, cols, pitch)
                assert (codes[:at] == 77).all() and (codes[at + rows * pitch:] == 77).all() and (got[:, cols:] == 77).all() and scales[rows] == 77


@pytest.mark.parametrize("dtype,x_type", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float32, torch.float32)])
@pytest.mark.parametrize("offset,pad", PLACES)
@pytest.mark.parametrize("post,gate", [(False, ""), (True, "token"), (False, "channel")])
def test_norm_block_wherever_rows_lie(ops, cuda, dtype, x_type, offset, pad, post, gate):
    """All outputs at once, between values that stay; weights at any multiple of four bytes."""
    eps, xs, ys = 1e-6, 0.9, 1.5
    for rows in (1, 3, 37):
        for width in WIDTHS:
            pitch = width + pad

            def window(dtype, content=None):
                buf = torch.full((offset + rows * pitch + 16,), 77.0, dtype=dtype, device="cuda")
                view = buf[offset:offset + rows * pitch].view(rows, pitch)[:, :width]
                if content is not None:
                    view.copy_(content)
                return buf, view
            x0, y0, pre, w, g0 = norm_inputs(rows, width, dtype, x_type, post, gate)
            _, x = window(x_type, x0)
            _, y = window(dtype, y0)
            g = window(dtype, g0)[1] if gate == "token" else g0
            pre = torch.cat([pre[:1], pre])[1:]
            x_buf, x_out = window(x_type)
            n_buf, n_out = window(dtype)
            codes, scales = torch.full((rows + 1, width + 5), 77, dtype=torch.int8, device="cuda"), torch.full((rows + 1,), 77.0, device="cuda")
            a = ops.NormArgs(rows, width, ops._Q8_DTYPES[dtype], ops._Q8_DTYPES[x_type], x.data_ptr(), pitch)
            a.d_y, a.ldy, a.x_scale, a.y_scale, a.eps = y.data_ptr(), pitch, xs, ys, eps
            a.d_post_w, a.d_pre_w = w.data_ptr() if post else None, pre.data_ptr()
            if gate:
                a.d_gate, a.ld_gate = g.data_ptr(), pitch if gate == "token" else 0
            a.d_x_out, a.ldx_out, a.d_out, a.ld_out = x_out.data_ptr(), pitch, n_out.data_ptr(), pitch
            a.d_codes, a.ld_codes, a.d_scales = codes.data_ptr(), width + 5, scales.data_ptr()
            assert ops.lib().b200attn_norm_block(C.byref(a), ops._current_stream()) == 0
            new, e_new, n, e_n, inv, e_inv = norm_reference(x, y, pre, w, g, False, xs, ys, eps)
            within(x_out, new, e_new, x_type)
            within(n_out, n, e_n, dtype)
            for buf, view in ((x_buf, x_out), (n_buf, n_out)):
                assert (buf[:offset] == 77).all() and (buf[offset + rows * pitch:] == 77).all() and (view.as_strided((rows, pad), (pitch, 1), offset + width) == 77).all()
            assert (codes[rows] == 77).all() and (codes[:, width:] == 77).all() and scales[rows] == 77
            if post:                          # a code is off by half a step and what 32 bits lose
                typed = n_out.double()
                assert ((codes[:rows, :width].double() * scales[:rows, None].double() - typed).abs() <= 0.51 * scales[:rows, None].double() + HALF_STEP[dtype] * typed.abs() + 1e-7).all()
            else:
                z = y.cpu().float() * (g.cpu().float() if gate else torch.tensor(1.0))
                want, s = define_codes((x.cpu().float() * torch.tensor(xs) + z * torch.tensor(ys)) * pre.cpu())
                assert torch.equal(codes[:rows, :width].cpu().double(), want), (rows, width)
                ideal = s.double().cuda() * inv[:, 0]
                within(scales[:rows], ideal, ideal.abs() * (e_inv[:, 0] + 3 * U), torch.float32)


@pytest.mark.parametrize("width", [3, 13, 64, 200, 256, 300])
def test_norm_block_of_many_short_rows(ops, cuda, width):
    x, y, pre, post, g = norm_inputs(20011, width, torch.bfloat16, torch.float32, True, "token")
    new, e_new, n, e_n, _, _ = norm_reference(x, y, pre, post, g, True, 1.0, 1.0, 1e-6)
    got_x, got_n = ops.norm_block(x, y, pre, post, g, True, out_dtype=torch.bfloat16)
    within(got_x, new, e_new, torch.float32)
    within(got_n, n, e_n, torch.bfloat16)
    want, s = define_codes(x)
    codes, scales = ops.quantize_rows(x)
    assert torch.equal(codes.cpu().double(), want) and torch.equal(scales.cpu(), s)


def test_norm_block_rows_out_of_the_ordinary(ops, cuda):
    x = activations(1, 5, 300, torch.float32)
    clean = ops.norm_block(x, out_dtype=torch.float32)[1]
    x[1, 7], x[3, 299] = float("nan"), float("inf")
    x[2] = 0
    _, n = ops.norm_block(x, out_dtype=torch.float32)
    assert torch.equal(n[[0, 4]], clean[[0, 4]]) and (n[2] == 0).all() and torch.isnan(n[1]).all()
    _, codes, scales = ops.norm_block(x)
    assert torch.isnan(scales[[1, 3]]).all() and (codes[1:4] == 0).all() and scales[2] == 0 and torch.isfinite(scales[[0, 4]]).all()


# ---- together, streams, graphs -------------------------------------------------------------------------------------------------------
def feed_forward(ops, gated, down, h, pre):
    """One feed-forward as a serving program runs it: norm to codes, gate / up, down onto the residual stream."""
    _, codes, scales = ops.norm_block(h, pre_w=pre, in_place=True)
    act = gated.forward_codes(codes, scales, out_dtype=torch.float16)
    return down.forward(act, out=h, accumulate=True)


def feed_forward_64(h, gate, up, down, pre):
    t = (h.cpu() * pre.cpu())
    codes, s = define_codes(t)
    inv = 1 / torch.sqrt(h.double().cpu().square().mean(1) + 1e-6)
    g, u = (product(codes, s.double() * inv, *define_codes(w)) for w in (gate, up))
    act = torch.nn.functional.silu(g) * u
    return act, h.double()


@pytest.mark.parametrize("rows", [1, 9, 16, 17, 128, 700])
def test_feed_forward(ops, cuda, rows):
    gate, up, down = (rand(s, *shape, std=0.03).bfloat16().cuda() for s, shape in ((1, (640, 256)), (2, (640, 256)), (3, (256, 640))))
    pre = (1 + rand(4, 256, std=0.1)).cuda()
    gated, lin = ops.Int8GatedLinear(gate, up), ops.Int8Linear(down)
    h = rand(5, rows, 256).cuda()
    act64, h64 = feed_forward_64(h, gate, up, down, pre)
    got = feed_forward(ops, gated, lin, h.clone(), pre)
    # From the exact activations on: they are rounded to fp16 (2^-11) and quantised (half a code, a / 254 per element), against which the rest is nothing.
    # The product's error is at most the sum over k of |error_k| |w_k|.
    wc, ws = define_codes(down)
    w = (wc * ws.double()[:, None]).cuda().abs()
    a = act64.abs().amax(1, keepdim=True)
    err = (act64.abs() * 2.0 ** -10 + a / 253.0) @ w.T
    want = h64 + act64 @ (wc * ws.double()[:, None]).cuda().T
    within(got, want, err + want.abs() * 8 * U, torch.float32)


def test_captured_feed_forward_and_another_stream(ops, cuda):
    gate, up, down = (rand(s, *shape, std=0.03).cuda() for s, shape in ((1, (384, 256)), (2, (384, 256)), (3, (256, 384))))
    pre = torch.ones(256, device="cuda")
    gated, lin = ops.Int8GatedLinear(gate, up), ops.Int8Linear(down)
    for rows in (1, 40, 300):
        starts = [rand(5 + i, rows, 256).cuda() for i in range(3)]
        want = [feed_forward(ops, gated, lin, h.clone(), pre) for h in starts]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for h, w in zip(starts, want):
                assert torch.equal(feed_forward(ops, gated, lin, h.clone(), pre), w)
            graphs, buffers = [], [torch.empty(rows, 256, device="cuda") for _ in range(2)]
            for buf in buffers:           # two graphs over the same weights, replayed side by side
                buf.copy_(starts[0])
                s.synchronize()
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=s):
                    feed_forward(ops, gated, lin, buf, pre)
                graphs.append(g)
        torch.cuda.synchronize()
        for i in range(3):
            streams = [torch.cuda.Stream() for _ in graphs]
            for j, (g, buf, st) in enumerate(zip(graphs, buffers, streams)):
                with torch.cuda.stream(st):
                    buf.copy_(starts[(i + j) % 3])
                    g.replay()
            torch.cuda.synchronize()
            for j, buf in enumerate(buffers):
                assert torch.equal(buf, want[(i + j) % 3])
    assert gated.device_status() == 0 and lin.device_status() == 0


def test_weights_given_again(ops, cuda):
    """A layer's weights may be replaced; strided weights are read as such."""
    big = rand(1, 80, 300).cuda()
    layer = ops.Int8Linear(big[:40, :200])
    x = activations(3, 21, 200, torch.float32)
    assert torch.equal(layer.forward(x), ops.Int8Linear(big[:40, :200].contiguous()).forward(x))
    other = big[40:, 100:300]
    ops._check(ops.lib().b200attn_q8_set_weights(layer.h, other.data_ptr(), None, ops.DTYPE_F32, 300, ops._current_stream()))
    assert torch.equal(layer.forward(x), ops.Int8Linear(other.contiguous()).forward(x))


# ---- offsets that pass 32 bits -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cols", [4096, 4099])
def test_rows_far_behind(ops, cuda, cols):
    """The last rows of matrices of more than 2^31 values, against the same rows by themselves."""
    rows, last = 2 ** 31 // 4096 + 77, 5
    x = torch.empty(rows, cols, dtype=torch.float16, device="cuda")
    x.zero_()
    x[-last:] = activations(3, last, cols, torch.float16)
    codes, scales = ops.quantize_rows(x)
    want, s = ops.quantize_rows(x[-last:].clone())
    assert torch.equal(codes[-last:], want) and torch.equal(scales[-last:], s) and (scales[:-last] == 0).all()
    del codes
    pre, post = (1 + rand(k, cols, std=0.1).cuda() for k in (4, 5))
    a, b = ops.norm_block(x, x, pre, post, out_dtype=torch.float16)
    wa, wb = ops.norm_block(x[-last:].clone(), x[-last:].clone(), pre, post, out_dtype=torch.float16)
    # another split of a row among threads sums its squares in another order: a root mean square off by 208 U of itself at most, so that a result is off by a rounding
    # of fp16 and what lies below it
    for got, ref in ((a, wa), (b, wb)):
        assert ((got[-last:].float() - ref.float()).abs() <= ref.float().abs() * 2.0 ** -10 + 2.0 ** -23).all()


@pytest.mark.parametrize("act", [-1, 1])
@pytest.mark.parametrize("y_type,out", [(torch.float16, 32768), (torch.float32, 32765)])
def test_results_far_behind(ops, cuda, act, y_type, out):
    rows, last = 2 ** 31 // 32768 + 300, 5
    ws = [rand(s, out, 64, std=0.05).cuda() for s in (5, 6)]
    layer = ops.Int8Linear(ws[0]) if act < 0 else ops.Int8GatedLinear(*ws, act)
    x = torch.zeros(rows, 64, device="cuda")
    x[-last:] = activations(3, last, 64, torch.float32)
    y = layer.forward(x, out_dtype=y_type)
    want = [product(*define_codes(x[-last:]), *define_codes(w)) for w in ws]
    if act < 0:
        within(y[-last:], want[0], PLAIN * want[0].abs(), y_type)
    else:
        within(y[-last:], glu_reference(*want, act), glu_bound(*want, act, y_type), y_type)
    assert not y[:-last].any() and layer.device_status() == 0


@pytest.mark.parametrize("rows", [3, 40])
def test_weights_far_behind(ops, cuda, rows):
    """More than 2^31 codes: the last columns against a layer of them alone."""
    out, last = 2 ** 31 // 8192 + 100, 64
    w = torch.zeros(out, 8192, dtype=torch.bfloat16, device="cuda")
    w[-last:] = rand(5, last, 8192, std=0.02).bfloat16().cuda()
    layer = ops.Int8Linear(w)
    x = activations(7, rows, 8192, torch.float16)
    y = layer.forward(x, out_dtype=torch.float32)
    assert torch.equal(y[:, -last:], ops.Int8Linear(w[-last:]).forward(x, out_dtype=torch.float32)) and not y[:, :-last].any()
    codes, scales = layer.weight_codes()
    want, s = define_codes(w[-last:])
    assert torch.equal(codes[-last:].cpu().double(), want) and torch.equal(scales[-last:].cpu(), s)
