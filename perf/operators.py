"""Block-scaled ("microscaled") operators: what they compute, on which sizes they are measured, and their plain forms.

A block-scaled tensor holds 32 consecutive elements of its last axis as 4-bit (E2M1) or 8-bit (E4M3) floating
point codes and one scale, a power of two in 8 bits (E8M0).  The scale is the smallest power of two under which
the block's largest magnitude fits the element type (6 for E2M1, 448 for E4M3), the elements are rounded to the
nearest, ties to even.  Kinds of cases:

  product     y = act(Q4(x) . W^T + b): the activations are quantised to 4 bits and multiplied by weights that are
              kept in 4 bits, as in a Linear layer that answers requests
  roundtrip   the values Q4(x) or Q8(x) stands for
  weights     dW = G^T . X8: the gradient of a Linear layer's weight from the 8-bit checkpoint of its input
  activation  dZ = G * act'(Z8): the gradient of an activation from the 8-bit checkpoint of its input

`own` false: elementary torch operations.  `own` true: the calls a user makes of this framework.

The framework launches on a stream of its own that torch's stream does not wait for, and `run` only enqueues, like a
program that keeps several passes in flight.  Whoever reads its results waits first: for the device, for `context()`, or
with the `finish` of the state's plan, which also raises what the kernels reported.
"""
import math

import torch

own = False

BLOCK = 32
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
# largest element as mantissa (in [0.5, 1)) and exponent; least normal exponent; mantissa bits
FORMATS = {"mx4": (0.75, 3, 0, 1), "mx8": (0.875, 9, -6, 3)}


# ---- cases -------------------------------------------------------------------------------------------------

def listed():
    return [
        # one request through a 4096-wide hidden layer: latency counts
        {"name": "product 1x4096x4096 bf16", "kind": "product", "rows": 1, "inner": 4096, "outer": 4096, "dtype": "bf16", "act": "relu"},
        # a few requests through the 784-wide first layer (24 blocks and a half)
        {"name": "product 16x784x4096 f32", "kind": "product", "rows": 16, "inner": 784, "outer": 4096, "dtype": "f32", "act": "relu"},
        # a classifier head on a ragged batch, odd contraction
        {"name": "product 203x4095x1000 f16", "kind": "product", "rows": 203, "inner": 4095, "outer": 1000, "dtype": "f16", "act": "none"},
        # a hidden layer at the inference batch of one GPU
        {"name": "product 8192x4096x4096 bf16", "kind": "product", "rows": 8192, "inner": 4096, "outer": 4096, "dtype": "bf16", "act": "relu"},
        # the same at the largest batch of the dense-layer benchmark
        {"name": "product 65536x4096x4096 bf16", "kind": "product", "rows": 65536, "inner": 4096, "outer": 4096, "dtype": "bf16", "act": "relu"},
        # quantising the weights of a hidden layer, and the hidden activations of a training batch
        {"name": "roundtrip mx4 1000x785 bf16", "kind": "roundtrip", "rows": 1000, "inner": 785, "dtype": "bf16", "format": "mx4"},
        {"name": "roundtrip mx8 65536x4096 f32", "kind": "roundtrip", "rows": 65536, "inner": 4096, "dtype": "f32", "format": "mx8"},
        # weight gradients: the small regression model, a hidden layer at one GPU's batch, the first layer at the whole one
        {"name": "weights 1024x32x128 f32", "kind": "weights", "rows": 1024, "inner": 32, "outer": 128, "dtype": "f32"},
        {"name": "weights 8192x4096x4096 f32", "kind": "weights", "rows": 8192, "inner": 4096, "outer": 4096, "dtype": "f32"},
        {"name": "weights 65536x784x4096 bf16", "kind": "weights", "rows": 65536, "inner": 784, "outer": 4096, "dtype": "bf16"},
        # activation gradients: a small odd batch, a hidden layer at the whole training batch
        {"name": "activation gelu 1023x129 bf16", "kind": "activation", "rows": 1023, "inner": 129, "dtype": "bf16", "act": "gelu"},
        {"name": "activation relu 65536x4096 f32", "kind": "activation", "rows": 65536, "inner": 4096, "dtype": "f32", "act": "relu"},
    ]


MOST_WORK = 65536 * 4096 * 4096


def draw(rng):
    def size(low, high):
        n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        return min(max(n, low), high)

    kind = rng.choice(["product", "product", "roundtrip", "weights", "weights", "activation"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if kind in ("product", "weights"):
        while True:
            rows, inner, outer = size(1, 65536), size(16, 8192), size(16, 8192)
            if rng.random() < 0.5:          # widths that networks have are multiples of something as often as not
                inner, outer = max(inner // 32 * 32, 32), max(outer // 16 * 16, 16)
            if rows * inner * outer <= MOST_WORK:
                break
        case = {"kind": kind, "rows": rows, "inner": inner, "outer": outer, "dtype": dtype}
        if kind == "product":
            case["act"] = rng.choice(["none", "relu", "silu", "gelu_tanh"])
        return case
    rows, inner = size(1, 65536), size(1, 4096)
    if rng.random() < 0.5:
        inner = max(inner // 32 * 32, 32)
    case = {"kind": kind, "rows": rows, "inner": inner, "dtype": dtype}
    if kind == "roundtrip":
        case["format"] = rng.choice(["mx4", "mx8"])
    else:
        case["act"] = rng.choice(["relu", "tanh", "sigmoid", "silu", "gelu_tanh", "gelu"])
    return case


def blocks(inner):
    return -(-inner // BLOCK)


def work(case):
    kind, r, k, width = case["kind"], case["rows"], case["inner"], BYTES[case["dtype"]]
    if kind == "product":
        n = case["outer"]
        return {"bytes": r * k * width + n * blocks(k) * 17 + n * width + r * n * width, "flops": 2.0 * r * k * n}
    if kind == "roundtrip":
        return {"bytes": 2 * r * k * width, "flops": 4.0 * r * k}
    if kind == "weights":
        n = case["outer"]
        return {"bytes": r * blocks(k) * 33 + r * n * width + n * k * 4, "flops": 2.0 * r * k * n}
    return {"bytes": r * blocks(k) * 33 + 2 * r * k * width, "flops": 8.0 * r * k}


# ---- plain forms -------------------------------------------------------------------------------------------

def quantize(x, fmt):
    """(elements under their scales, exponents of the scales) of x [rows, inner], in 32 bits; NaN for a block
    that holds an infinity or a NaN."""
    top, top_exponent, least, bits = FORMATS[fmt]
    rows, inner = x.shape
    padded = torch.nn.functional.pad(x.float(), (0, blocks(inner) * BLOCK - inner)).view(rows, -1, BLOCK)
    mantissa, exponent = torch.frexp(padded.abs().amax(-1))
    scale = (exponent - top_exponent + (mantissa > top).to(exponent.dtype)).clamp_min(-127)
    scale = torch.where(mantissa == 0, torch.full_like(scale, -127), scale)
    under = torch.ldexp(padded, -scale.unsqueeze(-1))
    step = torch.ldexp(torch.ones_like(under), (torch.frexp(under)[1] - 1).clamp_min(least) - bits)
    element = torch.round(under / step) * step
    return torch.where(torch.isfinite(padded).all(-1, keepdim=True), element, torch.full_like(element, math.nan)), scale


def stands_for(element, scale, inner):
    return torch.ldexp(element, scale.unsqueeze(-1)).flatten(1)[:, :inner]


def encode(element, scale, fmt):
    """The bytes of a block-scaled tensor: codes [rows, blocks * 16 or 32], scales [rows, blocks padded to a
    multiple of 4 with zeros]."""
    if fmt == "mx8":
        codes = element.flatten(1).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=element.device)
        code = torch.searchsorted(levels, element.abs().contiguous()).to(torch.uint8)
        code = (code | (torch.signbit(element).to(torch.uint8) << 3)).flatten(1)
        codes = code[:, 0::2] | (code[:, 1::2] << 4)
    return codes.contiguous(), torch.nn.functional.pad((scale + 127).to(torch.uint8), (0, -scale.shape[1] % 4)).contiguous()


def decode(codes, scales, fmt, inner):
    """The values (float32) a block-scaled tensor stands for."""
    if fmt == "mx8":
        element = codes.view(torch.float8_e4m3fn).float()
    else:
        levels = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
        code = torch.stack([codes & 15, codes >> 4], -1).flatten(1)
        element = torch.where(code >= 8, -levels[(code & 7).long()], levels[(code & 7).long()])
    return stands_for(element.view(codes.shape[0], -1, BLOCK), scales[:, :blocks(inner)].to(torch.int32) - 127, inner)


def activate(act, z):
    if act == "relu":
        return torch.clamp_min(z, 0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def slope(act, z):
    """act'(z)."""
    if act == "relu":
        return torch.where(torch.isnan(z), z, (z > 0).to(z.dtype))
    if act == "tanh":
        return 1 / torch.cosh(z.clamp(-40, 40)) ** 2
    if act == "sigmoid":
        return 1 / ((1 + torch.exp(-z)) * (1 + torch.exp(z)))
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z / (1 + torch.exp(z)))
    if act == "gelu_tanh":
        u = math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)
        t = torch.tanh(u)
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    return 0.5 * torch.erfc(-z / math.sqrt(2)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


# ---- inputs ------------------------------------------------------------------------------------------------

_context = None


def context():
    global _context
    if _context is None:
        from synaptik_b200 import native
        _context = native.Context(0)
    return _context


class Memory:
    """A framework buffer as memory that torch can see.  Every tensor over it keeps it alive; the last one frees it."""

    def __init__(self, nbytes):
        self.buffer = context().buffer(nbytes)
        self.__cuda_array_interface__ = {"data": (self.buffer.device_pointer(), False), "shape": (nbytes,), "typestr": "|u1", "version": 3}

    def tensor(self, shape, dtype):
        return torch.as_tensor(self, device="cuda").view(dtype).view(shape)

    def __del__(self):
        if hasattr(self, "buffer"):
            self.buffer.close()


class Plan:
    """A prepared program with its buffers, as a user's program keeps it."""

    def __init__(self, builder, inputs, outputs):
        from synaptik_b200 import native
        fed = [Memory(tensor.nbytes) for tensor in inputs]
        for memory, tensor in zip(fed, inputs):
            memory.tensor(tensor.shape, tensor.dtype).copy_(tensor)
        torch.cuda.synchronize()        # the framework's stream does not wait for torch's
        made = [Memory(math.prod(shape) * dtype.itemsize) for shape, dtype in outputs]
        self.results = [memory.tensor(*out) for memory, out in zip(made, outputs)]
        self.fed, self.inputs, self.outputs = fed, [m.buffer for m in fed], [m.buffer for m in made]
        self.executable = native.Executable(context(), builder.build())

    def __call__(self):
        self.executable.enqueue(self.inputs, self.outputs)
        return self.results

    def finish(self):
        """Waits for the enqueued passes; raises when a kernel reported an error."""
        self.executable.finish()

    def __del__(self):
        if hasattr(self, "executable"):
            try:
                self.finish()
            finally:
                self.executable.close()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, rows, inner, dtype = case["kind"], case["rows"], case["inner"], DTYPES[case["dtype"]]
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")      # noqa: E731
    state = {"case": dict(case)}
    if kind in ("product", "roundtrip"):
        # hidden activations: rows of different magnitude, a few features far above the others
        x = normal(rows, inner)
        x *= torch.exp(0.5 * normal(rows, 1))
        x *= torch.where(torch.rand(1, inner, generator=gen, device="cuda") < 0.01, 12.0, 1.0)
        state["x"] = x.to(dtype)
    if kind == "product":
        outer = case["outer"]
        bound = math.sqrt(6 / (inner + outer))
        weight = (2 * torch.rand(outer, inner, generator=gen, device="cuda") - 1) * bound
        state["codes"], state["scales"] = encode(*quantize(weight, "mx4"), "mx4")
        state["bias"] = (0.1 * normal(outer)).to(dtype)
    if kind == "weights":
        hidden = torch.clamp_min(normal(rows, inner), 0)       # what a ReLU passes on
        state["codes"], state["scales"] = encode(*quantize(hidden, "mx8"), "mx8")
        state["upstream"] = (normal(rows, case["outer"]) / rows).to(dtype) if case["dtype"] != "f16" else (0.01 * normal(rows, case["outer"])).to(dtype)
    if kind == "activation":
        state["codes"], state["scales"] = encode(*quantize(normal(rows, inner) * 2, "mx8"), "mx8")
        state["upstream"] = normal(rows, inner).to(dtype)
    if own:
        state["plan"] = own_plan(case, state)
    return state


def own_plan(case, state):
    from synaptik_b200 import program
    kind, rows, inner, dtype = case["kind"], case["rows"], case["inner"], DTYPES[case["dtype"]]
    g = program.GraphBuilder()
    storage = program.STORAGE_DTYPES[case["dtype"]]
    if kind == "product":
        x, w, b = g.feed(storage, (rows, inner)), g.mx_feed("mx4", (case["outer"], inner)), g.feed(storage, (case["outer"],))
        act = None if case["act"] == "none" else case["act"]
        g.publish(g.mx_linear(g.mx_quantize(x, "mx4"), w, b, act, storage))
        return Plan(g, [state["x"], state["codes"], state["scales"], state["bias"]], [((rows, case["outer"]), dtype)])
    if kind == "roundtrip":
        held = g.mx_quantize(g.feed(storage, (rows, inner)), case["format"])
        g.publish(g.mx_restore(held, storage))
        g.publish(held.codes)
        g.publish(held.scales)
        return Plan(g, [state["x"]], [((rows, inner), dtype), (held.codes.shape, torch.uint8), (held.scales.shape, torch.uint8)])
    held = g.mx_feed("mx8", (rows, inner))
    if kind == "weights":
        g.publish(g.mx_weight_gradient(held, g.feed(storage, (rows, case["outer"]))))
        return Plan(g, [state["codes"], state["scales"], state["upstream"]], [((case["outer"], inner), torch.float32)])
    g.publish(g.mx_activation_gradient(case["act"], held, g.feed(storage, (rows, inner))))
    return Plan(g, [state["codes"], state["scales"], state["upstream"]], [((rows, inner), dtype)])


def run(state):
    if own:
        return state["plan"]()[0]
    case = state["case"]
    kind, inner, dtype = case["kind"], case["inner"], DTYPES[case["dtype"]]
    if kind == "product":
        x = stands_for(*quantize(state["x"], "mx4"), inner)
        weight = decode(state["codes"], state["scales"], "mx4", inner)
        return activate(case["act"], x @ weight.T + state["bias"].float()).to(dtype)
    if kind == "roundtrip":
        return stands_for(*quantize(state["x"], case["format"]), inner).to(dtype)
    held = decode(state["codes"], state["scales"], "mx8", inner)
    if kind == "weights":
        return state["upstream"].float().T @ held
    return (state["upstream"].float() * slope(case["act"], held)).to(dtype)


# ---- the definition in 64 bits -----------------------------------------------------------------------------

def levels64(fmt):
    """Every non-negative value of the element type in ascending order: position = code without its sign."""
    exponent_bits, mantissa_bits, bias = (2, 1, 1) if fmt == "mx4" else (4, 3, 7)
    count = 8 if fmt == "mx4" else 127          # E4M3 has no infinity; its last code is NaN
    out = []
    for code in range(count):
        e, m = code >> mantissa_bits, code & ((1 << mantissa_bits) - 1)
        out.append(m * 2.0 ** (1 - bias - mantissa_bits) if e == 0 else (1 + m / 2.0 ** mantissa_bits) * 2.0 ** (e - bias))
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def quantized64(x, fmt):
    """The nearest value under the least power of two that holds the block, found among all values of the type."""
    levels = levels64(fmt)
    rows, inner = x.shape
    result = torch.zeros(rows, blocks(inner) * BLOCK, dtype=torch.float64, device=x.device)
    result[:, :inner] = x.double()
    result = result.view(-1, BLOCK)
    for at in range(0, result.shape[0], 1 << 19):
        part = result[at:at + (1 << 19)]
        largest = part.abs().max(-1, keepdim=True).values
        scale = torch.full_like(largest, 2.0 ** -127)
        wanted = largest / levels[-1]
        power = torch.exp2(torch.floor(torch.log2(wanted.clamp_min(2.0 ** -127))) - 1)
        for _ in range(3):                      # from below, until it holds
            power = torch.where(power < wanted, power * 2, power)
        scale = torch.maximum(scale, power)
        under = (part / scale).abs()
        above = torch.searchsorted(levels, under).clamp_max(len(levels) - 1)
        below = (above - 1).clamp_min(0)
        up, down = levels[above] - under, under - levels[below]
        take_up = (up < down) | ((up == down) & (above % 2 == 0))
        part.copy_(torch.where(take_up, levels[above], levels[below]) * torch.sign(part) * scale)
    return result.view(rows, -1)[:, :inner]


def held64(state, fmt, inner):
    codes, scales = state["codes"], state["scales"]
    if fmt == "mx4":
        codes = torch.stack((codes % 16, codes // 16), 2).reshape(codes.shape[0], -1)
        magnitude, negative = codes % 8, codes // 8
    else:
        magnitude, negative = codes % 128, codes // 128
    value = levels64(fmt)[magnitude.long()] * (1 - 2 * negative.double())
    return (value * torch.exp2(scales[:, :blocks(inner)].double() - 127).repeat_interleave(BLOCK, 1))[:, :inner]


def exact(case, seed):
    state = prepare(case, seed)
    kind, inner = case["kind"], case["inner"]
    if kind == "roundtrip":
        return quantized64(state["x"], case["format"])
    if kind == "product":
        z = quantized64(state["x"], "mx4") @ held64(state, "mx4", inner).T + state["bias"].double()
        if case["act"] == "relu":
            return torch.maximum(z, torch.zeros_like(z))
        if case["act"] == "silu":
            return z * torch.sigmoid(z)
        if case["act"] == "gelu_tanh":
            return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
        return z
    held = held64(state, "mx8", inner)
    upstream = state["upstream"].double()
    if kind == "weights":
        return upstream.T @ held
    if case["act"] == "relu":
        return torch.where(held > 0, upstream, torch.zeros_like(upstream))
    if case["act"] == "tanh":
        return upstream * (1 - torch.tanh(held) ** 2)
    if case["act"] == "sigmoid":
        return upstream * torch.sigmoid(held) * torch.sigmoid(-held)
    if case["act"] == "silu":
        return upstream * (torch.sigmoid(held) + held * torch.sigmoid(held) * torch.sigmoid(-held))
    if case["act"] == "gelu_tanh":
        u = 2 * math.sqrt(2 / math.pi) * (held + 0.044715 * held ** 3)
        return upstream * (torch.sigmoid(u) + held * torch.sigmoid(u) * torch.sigmoid(-u) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * held ** 2))
    return upstream * (torch.special.ndtr(held) + held * torch.exp(-held * held / 2) / math.sqrt(2 * math.pi))
