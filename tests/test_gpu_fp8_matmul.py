"""GPU: the FP8 matrix product and the projection on it.

Operands of small whole numbers with power-of-two scales have sums that FP32 holds exactly in any order, so those
products are compared bit by bit (BF16 results with the exact sum rounded once).  For other operands, with U = 2^-24 and
S the sum of the terms' magnitudes: a block's 128 products are exact, their FP32 sum is off by at most 2 U a term
(rounded or cut), a block's factor by U, each of the K/128 additions by U: (256 + K/128 + 2) U S in all."""
import pytest
import torch

from weftmoe_b200 import _lib
from weftmoe_b200.fp8 import (FP8Tensor, _quantize_fp8_both, fp8_linear, fp8_matmul, poll_fp8_matmul,
                              prepare_fp8_linear, quantize_fp8)

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
NAN_CODE = 0x7f


def generator(seed):
    return torch.Generator("cuda").manual_seed(seed)


def operand(rows, k, block_rows, seed, kind="whole", padding=NAN_CODE):
    """An FP8Tensor whose padding bytes are NaN: nothing behind k may be read."""
    g = generator(seed)
    kb = -(-k // 128)
    if kind == "whole":
        values = torch.randint(-4, 5, (rows, kb * 128), device="cuda", generator=g).float()
        scales = torch.exp2(torch.randint(-1, 2, (-(-rows // block_rows), kb), device="cuda", generator=g).float())
    else:
        values = (torch.randn(rows, kb * 128, device="cuda", generator=g) * 100).clamp(-448, 448)
        scales = torch.rand(-(-rows // block_rows), kb, device="cuda", generator=g) * 0.02 + 1e-3
    data = values.to(torch.float8_e4m3fn)
    data.view(torch.uint8)[:, k:] = padding
    return FP8Tensor(data, scales, (rows, k), block_rows)


def wide(t):
    rows, k = t.shape
    factor = t.scales.double().repeat_interleave(t.block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :k]
    return t.data[:, :k].double() * factor


def check(m, n, k, a_rows=1, b_rows=128, dtype=torch.float32, seed=0):
    a, b = operand(m, k, a_rows, seed), operand(n, k, b_rows, seed + 1)
    want = wide(a) @ wide(b).t()
    got = fp8_matmul(a, b, dtype=dtype)
    assert got.dtype == dtype and torch.equal(got, want.float().to(dtype)), (m, n, k)


@pytest.mark.parametrize("m", (1, 2, 15, 16, 17, 32, 33, 64, 65, 127, 128, 129, 255, 257))
@pytest.mark.parametrize("n, k", [(1, 1), (7, 128), (128, 129), (130, 1000), (256, 2049), (640, 384)])
def test_sizes(m, n, k):
    check(m, n, k)


@pytest.mark.parametrize("m, n, k", [(5, 300, 700), (40, 128, 4096), (130, 257, 1300), (300, 520, 640), (513, 770, 256)])
@pytest.mark.parametrize("a_rows, b_rows", [(1, 1), (1, 128), (128, 1), (128, 128)])
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
def test_blocks_and_types(m, n, k, a_rows, b_rows, dtype):
    check(m, n, k, a_rows, b_rows, dtype)


@pytest.mark.parametrize("b_rows", (1, 128))
@pytest.mark.parametrize("m, n, k", [(16, 256, 16384), (64, 2048, 2048), (100, 128, 8192), (1300, 2100, 130),
                                     (2500, 2900, 300), (1024, 4096, 1152), (4200, 520, 256), (2048, 2048, 2048), (8300, 8200, 250),
                                     (4100, 4197, 1100)])
def test_shared_tiles_and_long_grids(m, n, k, b_rows):
    """Tiles whose blocks several CTAs share, and grids of more tiles than there are SMs."""
    check(m, n, k, 1, b_rows)
    check(m, n, k, 1, b_rows, torch.bfloat16, seed=5)


@pytest.mark.parametrize("b_rows", (1, 128))
@pytest.mark.parametrize("blocks", (1, 4, 5, 8, 9, 31, 32, 33, 65))
def test_scales_on_the_tensor_cores(blocks, b_rows):
    """Large tiles with power-of-two scales, up to and beyond one group of 32 blocks and one of the packing kernel;
    a short last block; then the same with one scale that is no power of two, one zero and one NaN."""
    m, n = (1500, 1700) if blocks > 20 else (4100, 4200)   # large enough for pairs of SMs
    k = blocks * 128 - 5
    a, b = operand(m, k, 1, 50), operand(n, k, b_rows, 51)
    want = wide(a) @ wide(b).t()
    assert torch.equal(fp8_matmul(a, b, dtype=torch.float32), want.float())
    for value in (1.5, 0.0):
        b.scales[-1, -1] = value
        assert torch.equal(fp8_matmul(a, b, dtype=torch.float32), (wide(a) @ wide(b).t()).float())
    a.scales[77, 0] = float("nan")
    got = fp8_matmul(a, b)
    assert torch.isnan(got[77]).all() and not torch.isnan(got[:77]).any() and not torch.isnan(got[78:]).any()


def test_far_powers_of_two_on_the_tensor_cores():
    a, b = operand(4100, 1100, 1, 52), operand(4200, 1100, 128, 53)
    a.scales[:, 0], b.scales[:, 0] = 2.0 ** 100, 2.0 ** -101
    a.scales[:, 1], b.scales[:, 1] = 2.0 ** -60, 2.0 ** 62
    assert torch.equal(fp8_matmul(a, b, dtype=torch.float32), (wide(a) @ wide(b).t()).float())


@pytest.mark.parametrize("k", (4096, 16000))
def test_random_products_on_the_tensor_cores(k):
    """Quantised values: the accumulator cuts at most 2 U of what it holds at each of a group's 128 steps, so the bound of
    the general form holds here too.  In the mean square: a cut is U of the accumulator on average, always towards zero, and
    the accumulator of a group grows as the root of its steps (2/3 of its end on average): 128 * 2/3 * U = 2^-17.6."""
    a = quantize_fp8(torch.randn(1500, k, device="cuda", generator=generator(54)).bfloat16())
    b = quantize_fp8(torch.randn(1700, k, device="cuda", generator=generator(55)).bfloat16(), block_rows=128)
    want, terms = wide(a) @ wide(b).t(), wide(a).abs() @ wide(b).abs().t()
    got = fp8_matmul(a, b, dtype=torch.float32).double()
    assert ((got - want).abs() <= (256 + -(-k // 128) + 2) * U * terms).all()
    assert (got - want).norm() <= 2.0 ** -17.5 * want.norm()


@pytest.mark.parametrize("m, n, k", [(1, 512, 2048), (33, 700, 1100), (200, 300, 4097), (700, 1300, 2000),
                                     (2100, 4100, 2000)])
@pytest.mark.parametrize("a_rows, b_rows", [(1, 1), (1, 128), (128, 128)])
def test_any_scales(m, n, k, a_rows, b_rows):
    a, b = operand(m, k, a_rows, 3, "any"), operand(n, k, b_rows, 4, "any")
    want, terms = wide(a) @ wide(b).t(), wide(a).abs() @ wide(b).abs().t()
    bound = (256 + -(-k // 128) + 2) * U * terms
    got = fp8_matmul(a, b, dtype=torch.float32)
    assert ((got.double() - want).abs() <= bound).all()
    half = torch.finfo(torch.bfloat16).eps / 2
    assert ((fp8_matmul(a, b).double() - want).abs() <= bound + half * (want.abs() + bound)).all()
    assert torch.equal(fp8_matmul(a, b, dtype=torch.float32), got)


def test_far_scales():
    """Products of scales far from 1 that FP32 still holds; a zero scale; whole blocks of zeros."""
    a, b = operand(70, 512, 1, 6), operand(130, 512, 128, 7)
    a.scales[:, 0], b.scales[:, 0] = 2.0 ** 100, 2.0 ** -101
    a.scales[:, 1], b.scales[:, 1] = 2.0 ** -60, 2.0 ** 62
    a.scales[5], b.scales[:, 3] = 0.0, 0.0
    assert torch.equal(fp8_matmul(a, b, dtype=torch.float32), (wide(a) @ wide(b).t()).float())


@pytest.mark.parametrize("m", (20, 150))
def test_nan_stays_in_its_row(m):
    a, b = operand(m, 300, 1, 8), operand(140, 300, 128, 9)
    clean = fp8_matmul(a, b)
    a.scales[7, 1] = float("nan")
    a.data.view(torch.uint8)[11, 200] = NAN_CODE
    got = fp8_matmul(a, b)
    assert torch.isnan(got[[7, 11]]).all()
    rest = [r for r in range(m) if r not in (7, 11)]
    assert torch.equal(got[rest], clean[rest])


def test_empty_sizes():
    for m, n, k in ((0, 5, 128), (5, 0, 128), (5, 7, 0)):
        a, b = operand(m, k, 1, 1), operand(n, k, 128, 2)
        got = fp8_matmul(a, b)
        assert got.shape == (m, n) and not got.any()
    out = torch.ones(5, 9, device="cuda")
    fp8_matmul(operand(5, 0, 1, 1), operand(7, 0, 128, 2), dtype=torch.float32, out=out[:, 1:8])
    assert not out[:, 1:8].any() and (out[:, [0, 8]] == 1).all()


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("m, n", [(3, 65), (40, 128), (130, 200), (300, 512), (4100, 4200)])
@pytest.mark.parametrize("left, right", [(8, 8), (1, 2), (0, 3)])
def test_out_is_a_slice(m, n, left, right, dtype):
    """Rows of a wider tensor, aligned or not: every element beside the slice stays."""
    a, b = operand(m, 640, 1, 10), operand(n, 640, 128, 11)
    holder = torch.full((m + 2, left + n + right), 7.0, dtype=dtype, device="cuda")
    view = holder[1:-1, left:left + n]
    assert fp8_matmul(a, b, dtype=dtype, out=view) is view
    assert torch.equal(view, (wide(a) @ wide(b).t()).float().to(dtype))
    view.fill_(7.0)
    assert (holder == 7).all()


def test_a_written_out_is_a_change_in_place():
    a, b = operand(9, 128, 1, 3), operand(40, 128, 128, 4)
    out = torch.zeros(9, 40, device="cuda")
    leaf = torch.ones(9, 40, device="cuda", requires_grad=True)
    product = leaf * out                                          # keeps out for its gradient
    fp8_matmul(a, b, dtype=torch.float32, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.sum().backward()
    with torch.inference_mode():
        out = torch.zeros(9, 40, device="cuda")
        assert torch.equal(fp8_matmul(a, b, dtype=torch.float32, out=out), fp8_matmul(a, b, dtype=torch.float32))


def test_linear_entry_of_an_empty_sum():
    out = torch.full((5, 8), 7.0, device="cuda", dtype=torch.bfloat16)
    code = _lib.load().wm_fp8_linear(None, 0, 5, 0, None, None, 8, out.data_ptr(), None, 0,
                                     torch.cuda.current_stream().cuda_stream)
    assert code == _lib.WM_OK and not out.any()


@pytest.mark.parametrize("m, n, k", [(9, 200, 512), (200, 300, 512), (600, 1100, 256), (64, 256, 8192), (4100, 4200, 640)])
def test_accumulate(m, n, k):
    a, b = operand(m, k, 1, 12), operand(n, k, 1, 13)
    out = torch.randint(-100, 100, (m, n), device="cuda", generator=generator(14)).float()
    want = out.double() + 2 * (wide(a) @ wide(b).t())
    for _ in range(2):
        fp8_matmul(a, b, dtype=torch.float32, out=out, accumulate=True)
    assert torch.equal(out, want.float())


def test_refusals():
    a, b = operand(8, 256, 1, 1), operand(16, 256, 128, 2)
    with pytest.raises(ValueError, match="same device"):
        fp8_matmul(a, operand(16, 384, 128, 2))
    with pytest.raises(ValueError, match="dtype"):
        fp8_matmul(a, b, dtype=torch.float16)
    with pytest.raises(ValueError, match="accumulation"):
        fp8_matmul(a, b, accumulate=True, out=torch.zeros(8, 16, dtype=torch.bfloat16, device="cuda"))
    for out in (torch.zeros(8, 15, device="cuda"), torch.zeros(16, 8, device="cuda").t(),
                torch.zeros(1, 16, device="cuda").expand(8, 16), torch.zeros(8, 16)):
        with pytest.raises(ValueError, match="mismatch"):
            fp8_matmul(a, b, dtype=torch.float32, out=out)


def test_captured_twice_and_on_another_stream():
    a, b = operand(48, 1024, 1, 15), operand(1024, 1024, 128, 16)
    big = operand(900, 1024, 1, 17)
    want, want_big = fp8_matmul(a, b), fp8_matmul(big, b)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append((fp8_matmul(a, b), fp8_matmul(big, b)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for graph, stream in zip(graphs, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for small, large in outs:
        assert torch.equal(small, want) and torch.equal(large, want_big)
    poll_fp8_matmul()


@pytest.mark.parametrize("m", (16, 1500))
def test_captured_behind_copies_clears_and_joins(m):
    """A product may start its prologue under the kernel before it: here what is before it is a memory copy, a clear,
    another stream's work, or a kernel that writes its operands."""
    host = torch.randn(m, 1024).bfloat16().pin_memory()
    x = torch.empty(m, 1024, device="cuda", dtype=torch.bfloat16)
    w = quantize_fp8(torch.randn(1700, 1024, device="cuda").bfloat16(), block_rows=128)
    out = torch.empty(m, 1700, device="cuda")
    side = torch.cuda.Stream()

    def step():
        x.copy_(host, non_blocking=True)
        a = quantize_fp8(x)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = fp8_matmul(a, w)
        out.zero_()
        fp8_matmul(a, w, dtype=torch.float32, out=out, accumulate=True)
        torch.cuda.current_stream().wait_stream(side)
        fp8_matmul(a, w, dtype=torch.float32, out=out, accumulate=True)
        return other

    side.wait_stream(torch.cuda.current_stream())
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other = step()
    for seed in (1, 2):
        host.copy_(torch.randn(m, 1024, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        a = quantize_fp8(host.cuda())
        once = fp8_matmul(a, w, dtype=torch.float32)
        assert torch.equal(out, 2 * once) and torch.equal(other, fp8_matmul(a, w))
    del graph


def test_offsets_beyond_32_bits():
    rows, k = 66000, 32768                                       # 2.2 GB of weights
    b = FP8Tensor(torch.zeros(rows, k, dtype=torch.float8_e4m3fn, device="cuda"),
                  torch.ones(-(-rows // 128), k // 128, device="cuda"), (rows, k), 128)
    b.data[-1] = 1.0
    a = operand(3, k, 1, 18)
    got = fp8_matmul(a, b, dtype=torch.float32)
    assert torch.equal(got[:, -1], wide(a).sum(1).float()) and not got[:, :-1].any()
    del b
    m, n = 70000, 32768                                          # 2.3 G elements of the result
    a, b = operand(m, 128, 1, 19), operand(n, 128, 128, 20)
    got = fp8_matmul(a, b)
    assert torch.equal(got[-5:], (wide(a)[-5:] @ wide(b).t()).float().bfloat16())
    assert torch.equal(got[:5], (wide(a)[:5] @ wide(b).t()).float().bfloat16())


# ------------------------------------------------------------------ quantising both ways
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("rows, cols", [(1, 8), (1, 1), (127, 128), (128, 136), (129, 264), (300, 77), (1000, 520)])
def test_both_ways_at_once_are_the_two_ways(rows, cols, dtype):
    x = torch.randn(rows, cols, device="cuda", generator=generator(30)).to(dtype)
    x[0, 0], x[rows // 2, cols // 2] = 3e38, 0.0
    x[:, cols // 3] = 0.0
    if rows > 100:
        x[100, 3], x[rows - 1, cols - 1] = float("nan"), float("inf")
    for source in (x, torch.cat([x, x])[rows:], x.new_empty(rows * cols + 1)[1:].view(rows, cols).copy_(x)):
        straight, flipped = _quantize_fp8_both(source)
        # the plain definition on both: by way of the FP32 source, whose kernel is another one
        for got, want in ((straight, quantize_fp8(x.float())), (flipped, quantize_fp8(x.float(), transpose=True)),
                          (flipped, quantize_fp8(source, transpose=True))):
            assert got.shape == want.shape and got.block_rows == want.block_rows == 1
            assert torch.equal(got.data.view(torch.uint8), want.data.view(torch.uint8))
            assert torch.equal(got.scales.view(torch.int32), want.scales.view(torch.int32))


def test_both_ways_of_several_matrices():
    x = torch.randn(3, 200, 256, device="cuda", generator=generator(31)).bfloat16()
    straight, flipped = _quantize_fp8_both(x)
    for e in range(3):
        assert torch.equal(straight.matrix(e).dequantize(), quantize_fp8(x[e]).dequantize())
        assert torch.equal(flipped.matrix(e).dequantize(), quantize_fp8(x[e], transpose=True).dequantize())


# ------------------------------------------------------------------ the projection
def held(x, **how):
    return wide(quantize_fp8(x, **how))


def product_close(got, left, right, what):
    want, terms = left @ right.t(), left.abs() @ right.abs().t()
    bound = (256 + -(-left.shape[1] // 128) + 2) * U * terms
    bound = bound + torch.finfo(got.dtype).eps / 2 * (want.abs() + bound)
    assert ((got.double() - want).abs() <= bound).all(), what


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("tokens, inputs, outputs", [(1, 128, 256), (3, 100, 77), (64, 640, 256), (129, 384, 130),
                                                     (1000, 512, 1024)])
def test_linear_and_gradients(tokens, inputs, outputs, dtype):
    g = generator(21)
    x = torch.randn(tokens, inputs, device="cuda", generator=g).to(dtype).requires_grad_()
    weight = (torch.randn(outputs, inputs, device="cuda", generator=g) / 16).to(dtype).requires_grad_()
    dy = torch.randn(tokens, outputs, device="cuda", generator=g).to(dtype)
    y = fp8_linear(x, weight, prepare_fp8_linear(weight))
    dx, dweight = torch.autograd.grad(y, (x, weight), dy)
    assert y.dtype == dx.dtype == dweight.dtype == dtype
    w = held(weight.detach(), block_rows=128)
    product_close(y, held(x.detach()), w, "y")
    product_close(dx, held(dy), w.t(), "dx")
    product_close(dweight, held(dy, transpose=True), held(x.detach(), transpose=True), "dweight")
    with torch.no_grad():
        assert torch.equal(fp8_linear(x, weight, prepare_fp8_linear(weight, training=False)), y)
    shaped = fp8_linear(x.detach().view(1, tokens, inputs), weight, prepare_fp8_linear(weight))
    assert shaped.shape == (1, tokens, outputs) and torch.equal(shaped[0], y)


def test_linear_gradient_against_differences():
    """x and W on a grid that E4M3 holds exactly: y is then linear in each, and differences are exact."""
    g = generator(22)
    x = torch.randint(-6, 7, (5, 256), device="cuda", generator=g).float()
    weight = torch.randint(-6, 7, (130, 256), device="cuda", generator=g).float()
    x[:, ::128] = 12.0                       # the same largest value, so the same scale, in every block
    weight[:, ::128] = 12.0
    dy = torch.zeros(5, 130, device="cuda")
    dy[2, 77] = 1.0
    leaves = x.clone().requires_grad_(), weight.clone().requires_grad_()
    y = fp8_linear(*leaves, prepare_fp8_linear(leaves[1]))
    dx, dweight = torch.autograd.grad(y, leaves, dy)
    run = lambda x, w: fp8_linear(x, w, prepare_fp8_linear(w))[2, 77].item()
    for at in (1, 130, 255):
        moved = x.clone()
        moved[2, at] += 1
        assert run(moved, weight) - run(x, weight) == dx[2, at].item()
        moved = weight.clone()
        moved[77, at] += 1
        assert run(x, moved) - run(x, weight) == dweight[77, at].item()
    assert not dx[[0, 1, 3, 4]].any() and dweight[77].any() and not dweight[:77].any()


def test_linear_of_no_tokens_and_of_broadcast_inputs():
    weight = torch.randn(96, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    prepared = prepare_fp8_linear(weight)
    x = torch.zeros(0, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    dx, dweight = torch.autograd.grad(fp8_linear(x, weight, prepared).sum(), (x, weight))
    assert dx.shape == (0, 256) and not dweight.any()
    row = torch.randn(1, 256, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = fp8_linear(row.expand(4, 256), weight, prepared)
    dy = torch.randn(4, 96, device="cuda", dtype=torch.bfloat16)
    dx, = torch.autograd.grad(y, row, dy)
    each = fp8_matmul(quantize_fp8(dy), prepared.weight_t).double()
    assert ((dx.double() - each.sum(0)).abs() <= 4 * 2.0 ** -8 * each.abs().sum(0)).all()   # torch's BF16 sum of 4
    y = fp8_linear(row, weight, prepared)
    torch.autograd.grad(y.sum(), (row, weight))                                             # an expanded dy


def test_linear_refuses_weights_of_another_version():
    weight = torch.randn(64, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    x = torch.randn(4, 128, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    prepared = prepare_fp8_linear(weight)
    with pytest.raises(ValueError, match="different parameters"):
        fp8_linear(x, weight.detach().clone(), prepared)
    with pytest.raises(ValueError, match="training=True"):
        fp8_linear(x, weight, prepare_fp8_linear(weight, training=False))
    with pytest.raises(ValueError, match="match"):
        fp8_linear(x[:, :64], weight, prepared)
    y = fp8_linear(x, weight, prepared)
    with torch.no_grad():
        weight.mul_(2)
    with pytest.raises(RuntimeError, match="stale"):
        fp8_linear(x, weight, prepared)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    prepared.weight.scales.mul_(2)
    with pytest.raises(RuntimeError, match="modified"):
        fp8_linear(x, weight, prepared)


def test_linear_takes_an_imported_weight():
    weight = operand(130, 300, 128, 23, "any", padding=0)
    parameter = torch.zeros(130, 300, device="cuda", dtype=torch.bfloat16)
    x = torch.randn(70, 300, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    prepared = prepare_fp8_linear(weight)
    y = fp8_linear(x, parameter, prepared)
    product_close(y, held(x.detach()), wide(weight), "y")
    dy = torch.randn(70, 130, device="cuda", dtype=torch.bfloat16)
    dx, = torch.autograd.grad(y, x, dy)
    product_close(dx, held(dy), wide(weight).t(), "dx")


def test_captured_training_step_of_a_projection():
    weight = torch.randn(256, 384, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    prepared = prepare_fp8_linear(weight)
    x = torch.randn(200, 384, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    dy = torch.randn(200, 256, device="cuda", dtype=torch.bfloat16)

    def step():
        y = fp8_linear(x, weight, prepared)
        return (y.detach(), *torch.autograd.grad(y, (x, weight), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        x.copy_(torch.randn(200, 384, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, step()))
