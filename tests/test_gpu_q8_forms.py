"""GPU: the kernels of the 8-bit operators that rows of a call choose by their number, width and place, each reached on purpose; their statistics; what they write to."""
import pytest
import torch

from test_gpu_q8 import TYPES, U, activations, define_codes, norm_inputs, norm_reference, rand, within

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def many(torch_, width):
    """More rows than a thread per eight values has under way at once on this device: a warp then holds a row."""
    sms = torch_.cuda.get_device_properties(0).multi_processor_count
    return sms * (1024 // max(64, (width // 8 + 31) // 32 * 32)) + 7


# 264 .. 512: two eights a lane, 520 .. 1024: four
@pytest.mark.parametrize("width", [264, 400, 512, 520, 776, 1000, 1024])
@pytest.mark.parametrize("dtype,x_type", [(BF16, F32), (F16, F16), (BF16, BF16), (F32, F32), (F16, F32)])
@pytest.mark.parametrize("post,gate,xs,ys", [(False, "", 1.0, 1.0), (True, "sigmoid", 1.0, 0.25), (False, "channel", 0.9, 1.5), (True, "token", 0.5, -1.0)])
def test_norm_block_of_many_rows(ops, cuda, width, dtype, x_type, post, gate, xs, ys):
    x, y, pre, post, g = norm_inputs(many(cuda, width), width, dtype, x_type, post, gate)
    sigmoid = gate == "sigmoid"
    new, e_new, n, e_n, inv, e_inv = norm_reference(x, y, pre, post, g, sigmoid, xs, ys, 1e-6)
    got_x, got_n = ops.norm_block(x, y, pre, post, g, sigmoid, xs, ys, out_dtype=dtype)
    within(got_x, new, e_new, x_type)
    within(got_n, n, e_n, dtype)
    kept = x.clone()
    _, codes, scales = ops.norm_block(kept, y, pre, post, g, sigmoid, xs, ys, in_place=True)
    assert torch.equal(kept, got_x)
    if post is None:
        z = y.cpu().float() if g is None else y.cpu().float() * g.cpu().float()
        want, s = define_codes((x.cpu().float() * torch.tensor(xs) + z * torch.tensor(ys)) * pre.cpu())
        assert torch.equal(codes.cpu().double(), want)
        ideal = s.double().cuda() * inv[:, 0]
        within(scales, ideal, ideal.abs() * (e_inv[:, 0] + 3 * U), F32)
    else:
        # a code is off by half a step and what 32 bits lose
        err = (codes.double() * scales[:, None].double() - n).abs()
        assert (err <= 0.51 * scales[:, None].double() + e_n + 1e-30).all()


@pytest.mark.parametrize("width", [264, 512, 520, 1024])
@pytest.mark.parametrize("dtype,x_type", [(F16, F32), (BF16, BF16), (F32, F32)])
def test_norm_of_many_rows_without_a_block_output(ops, cuda, width, dtype, x_type):
    rows = many(cuda, width)
    x, pre = activations(11, rows, width, x_type), (1 + rand(17, width, std=0.1)).cuda()
    got_x, codes, scales = ops.norm_block(x, pre_w=pre)
    want, s = define_codes(x.cpu().float() * pre.cpu())
    assert torch.equal(got_x, x) and torch.equal(codes.cpu().double(), want)
    ideal = s.double().cuda() / torch.sqrt(x.double().square().mean(1) + 1e-6)
    within(scales, ideal, ideal.abs() * 27 * U, F32)          # the root mean square as below (45 / 2 + 1), the quotient
    _, _, n, e_n, _, _ = norm_reference(x, None, pre, None, None, False, 1.0, 1.0, 1e-6)
    within(ops.norm_block(x, pre_w=pre, out_dtype=dtype)[1], n, e_n, dtype)


@pytest.mark.parametrize("rows,width,pad", [(1, 8, 0), (5, 64, 0), (3, 1000, 0), (2500, 512, 0), (1500, 1024, 0), (7, 1024, 0), (9, 2050, 0), (40, 4096, 0), (3, 4099, 1), (2, 8192, 0), (3, 8200, 0), (2, 16384, 0),
                                            (2, 16377, 0), (3, 20001, 0), (2, 33000, 0), (1, 49152, 0), (3, 500, 3), (2, 10000, 5)])
def test_root_mean_squares(ops, cuda, rows, width, pad):
    """Squares of the same sign, so that errors of a sum are all there is.  A thread adds at most 32 of them (rows of more than about 16384 values: one in 512 of the row) one
    after the other and a tree of ten steps joins the threads; each addition rounds once, so do the last product in front of it, the mean and the sum with eps.  The root has half of
    that and a rounding, quotient and product one each."""
    x = activations(3, rows, width, F32, width + pad if pad else None)
    own = 32 if width <= 16377 else max(32, -(-width // 512))
    n = ops.norm_block(x, out_dtype=F32)[1]
    want = x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + 1e-6)
    within(n, want, want.abs() * ((own + 10 + 3) / 2 + 3) * U, F32)


# aligned rows that one warp holds in eight groups a lane, some of them empty
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [1032, 1224, 1536, 2040, 2048])
@pytest.mark.parametrize("rows", [1, 6, 1001])
def test_quantize_by_a_warp(ops, cuda, dtype, cols, rows):
    x = activations(rows + cols, rows, cols, dtype)
    if rows > 5:
        x[1], x[2, cols - 1], x[3, 0] = 0, float("inf"), float("nan")
    want, s = define_codes(x)
    codes, scales = ops.quantize_rows(x)
    assert torch.equal(codes.cpu().double(), want)
    assert torch.equal(torch.nan_to_num(scales.cpu(), nan=-7.0), torch.nan_to_num(s, nan=-7.0))
    wide = torch.full((rows + 2, cols + 16), 77, dtype=torch.int8, device="cuda")
    assert ops.lib().b200attn_q8_quantize(x.data_ptr(), ops._Q8_DTYPES[dtype], cols, rows, cols, wide[1:].data_ptr(), cols + 16, scales.data_ptr(), ops._current_stream()) == 0
    assert torch.equal(wide[1:rows + 1, :cols], codes) and (wide[0] == 77).all() and (wide[rows + 1] == 77).all() and (wide[:, cols:] == 77).all()
