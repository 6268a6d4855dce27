"""Block-scaled operations where positions, bytes or results pass 2^31 and 2^32, through the C ABI.  Inputs are made and results
compared on the device."""
import numpy as np
import pytest

import mx_reference as ref
from synaptik_b200 import native, program
from synaptik_b200.program import BF16, F32, GraphBuilder

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ctx():
    c = native.Context(0)
    yield c
    c.close()


class Device:
    """Buffers of a test, seen by torch, released at its end."""

    def __init__(self, ctx):
        self.ctx, self.buffers = ctx, []

    def empty(self, shape, dtype):
        count = int(np.prod(shape)) * dtype.itemsize
        buffer = self.ctx.buffer(count)
        self.buffers.append(buffer)
        holder = type("Memory", (), {"__cuda_array_interface__": {"data": (buffer.device_pointer(), False), "shape": (count,), "typestr": "|u1", "version": 3}})()
        return buffer, torch.as_tensor(holder, device="cuda").view(dtype).view(shape)

    def run(self, builder, inputs, outputs):
        torch.cuda.synchronize()
        exe = native.Executable(self.ctx, builder.build())
        try:
            exe.run(inputs, outputs)
        finally:
            exe.close()


@pytest.fixture
def device(ctx):
    d = Device(ctx)
    yield d
    ctx.synchronize()
    for b in d.buffers:
        b.close()
    torch.cuda.empty_cache()


ROWS = (1 << 27) + 37           # rows of one word of scales: groups of eight elements pass 2^31, bytes of 8-bit codes 2^32


@pytest.mark.parametrize("cols", [1, 16])
@pytest.mark.parametrize("fmt", ["mx4", "mx8"])
def test_element_wise_passes_over_many_rows(device, fmt, cols):
    codes_width = program.mx_code_bytes(fmt, cols)
    x_buffer, x = device.empty((ROWS, cols), torch.bfloat16)
    c_buffer, codes = device.empty((ROWS, codes_width), torch.uint8)
    s_buffer, scales = device.empty((ROWS, 4), torch.uint8)
    y_buffer, y = device.empty((ROWS, cols), torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(cols)
    period = torch.randn((1 << 20) + 7, cols, generator=gen, device="cuda").to(torch.bfloat16)
    for at in range(0, ROWS, period.shape[0]):
        part = x[at:at + period.shape[0]]
        part.copy_(period[:part.shape[0]])
    codes.fill_(255), scales.fill_(255)
    g = GraphBuilder()
    xv = g.feed(BF16, (ROWS, cols))
    held = g.mx_quantize(xv, fmt)
    g.publish(held.codes)
    g.publish(held.scales)
    g.publish(g.mx_restore(held, BF16))
    device.run(g, [x_buffer], [c_buffer, s_buffer, y_buffer])
    want_codes, want_scales = ref.quantize(period.float().cpu().numpy().astype(np.float64), fmt)
    want = torch.from_numpy(ref.values(want_codes, want_scales, fmt, cols)).to("cuda", torch.bfloat16)
    want_codes, want_scales = torch.from_numpy(want_codes).cuda(), torch.from_numpy(want_scales).cuda()
    for at in range(0, ROWS, period.shape[0]):
        here = slice(at, min(at + period.shape[0], ROWS))
        n = here.stop - at
        assert torch.equal(codes[here], want_codes[:n]) and torch.equal(scales[here], want_scales[:n]) and torch.equal(y[here], want[:n]), at
    if fmt == "mx8":            # the gradient of a ReLU, the tensor itself as upstream
        g = GraphBuilder()
        held, up = g.mx_feed("mx8", (ROWS, cols)), g.feed(BF16, (ROWS, cols))
        g.publish(g.mx_activation_gradient("relu", held, up))
        device.run(g, [c_buffer, s_buffer, x_buffer], [y_buffer])
        want = torch.where(want > 0, period, torch.zeros_like(period))
        for at in range(0, ROWS, period.shape[0]):
            here = slice(at, min(at + period.shape[0], ROWS))
            assert torch.equal(y[here], want[:here.stop - at]), at


@pytest.mark.parametrize("k,n", [(64, 4096), (16384, 160), (96, 4091)])
def test_product_past_32_bits(device, k, n):
    """More than 2^31 results, or more than 2^32 bytes of codes: rows from all over against a product of those rows alone."""
    rows = 600_011
    rng = np.random.default_rng(k)
    w = ref.quantize(rng.standard_normal((n, k)), "mx4")
    x_buffer, x = device.empty((rows, k // 2), torch.uint8)
    s_buffer, xs = device.empty((rows, program.mx_scale_bytes(k)), torch.uint8)
    y_buffer, y = device.empty((rows, n), torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(k)
    x.random_(0, 256, generator=gen)
    xs.random_(120, 128, generator=gen)
    wb, ws = device.ctx.upload(w[0]), device.ctx.upload(w[1])
    device.buffers += [wb, ws]

    def graph(m):
        g = GraphBuilder()
        g.publish(g.mx_linear(g.mx_feed("mx4", (m, k)), g.mx_feed("mx4", (n, k)), None, "relu", BF16))
        return g
    device.run(graph(rows), [x_buffer, s_buffer, wb, ws], [y_buffer])
    m = 20000                   # enough for the same tiles
    some_x, sx = device.empty((m, k // 2), torch.uint8)
    some_s, ss = device.empty((m, xs.shape[1]), torch.uint8)
    some_y, sy = device.empty((m, n), torch.bfloat16)
    for first in (0, rows // 2 + 3, rows - m):
        sx.copy_(x[first:first + m])
        ss.copy_(xs[first:first + m])
        device.run(graph(m), [some_x, some_s, wb, ws], [some_y])
        assert torch.equal(sy, y[first:first + m]), first
    xv = ref.values(x[-5:].cpu().numpy(), xs[-5:].cpu().numpy(), "mx4", k)
    wv = ref.values(*w, "mx4", k)
    want, s = np.maximum(xv @ wv.T, 0), np.abs(xv) @ np.abs(wv).T
    got = y[-5:].float().cpu().numpy()
    assert (np.abs(got - want) <= (k / 32 + 4) * 2.0 ** -23 * s + 2.0 ** -8 * 1.01 * want).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weight_gradient_past_32_bits(device, dtype):
    """More than 2^31 elements of the gradient.  Each of 586 or more partial sums (1024 rows at most) loses up to 64 units of
    2^-23 of itself, about 32 standard deviations of a term; the results are about 775 of them: 2e-4 of the norm at the most."""
    rows, n, k = 600_011, 4096, 32
    g_buffer, up = device.empty((rows, n), dtype)
    c_buffer, codes = device.empty((rows, 32), torch.uint8)
    s_buffer, scales = device.empty((rows, 4), torch.uint8)
    d_buffer, dw = device.empty((n, k), torch.float32)
    gen = torch.Generator(device="cuda").manual_seed(1)
    up.normal_(generator=gen)
    held = torch.randn(rows, 32, generator=gen, device="cuda").to(torch.float8_e4m3fn)
    codes.copy_(held.view(torch.uint8))
    scales.zero_()
    scales[:, 0].random_(125, 129, generator=gen)
    g = GraphBuilder()
    g.publish(g.mx_weight_gradient(g.mx_feed("mx8", (rows, k)), g.feed(BF16 if dtype == torch.bfloat16 else F32, (rows, n))))
    device.run(g, [c_buffer, s_buffer, g_buffer], [d_buffer])
    x = held.double() * torch.exp2(scales[:, :1].double() - 127)
    want = torch.zeros(n, k, dtype=torch.float64, device="cuda")
    for at in range(0, rows, 50_000):
        want += up[at:at + 50_000].double().T @ x[at:at + 50_000]
    assert (dw.double() - want).norm() <= 2e-4 * want.norm()
