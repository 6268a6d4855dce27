"""Block-scaled tensors without a GPU: the reference implementation against itself, plans, refusals."""
import struct

import numpy as np
import pytest

import mx_reference as ref
from synaptik_b200 import native, program
from synaptik_b200.program import BF16, F16, F32, I32, U8, GraphBuilder


@pytest.mark.parametrize("fmt", ["mx4", "mx8"])
def test_reference_rounds_to_the_nearest_and_never_saturates(fmt):
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((40, 100)) * np.exp2(rng.integers(-30, 30, (40, 1)))).astype(np.float32)
    codes, scales = ref.quantize(x, fmt)
    assert codes.shape == (40, program.mx_code_bytes(fmt, 100)) and scales.shape == (40, program.mx_scale_bytes(100))
    back = ref.values(codes, scales, fmt, 100)
    top = ref.levels(fmt)[-1]
    scale = np.repeat(np.exp2(scales[:, :4].astype(float) - 127), 32, 1)[:, :100]
    assert (np.abs(x) <= top * scale).all()
    # half a step: relative above the smallest normal element, absolute below
    half = {"mx4": (2.0 ** -2, 0.25), "mx8": (2.0 ** -4, 2.0 ** -10)}[fmt]
    assert (np.abs(back - x) <= np.maximum(half[0] * np.abs(x), half[1] * scale)).all()
    again = ref.quantize(back, fmt)
    assert np.array_equal(ref.values(*again, fmt, 100), back)


def test_reference_zero_and_non_finite_blocks():
    x = np.zeros((1, 96), dtype=np.float32)
    x[0, 40], x[0, 70] = np.inf, np.nan
    codes, scales = ref.quantize(x, "mx8")
    assert scales.tolist() == [[0, 255, 255, 0]] and not codes.any()
    assert np.isnan(ref.values(codes, scales, "mx8", 96)[0, 32:]).all()


def test_plan_of_every_operation():
    g = GraphBuilder()
    x, gate = g.feed(F32, (2, 50, 100)), g.feed(F32, (2, 50, 40))
    held = g.mx_quantize(x, "mx8")
    g.publish(g.mx_weight_gradient(held, gate))
    g.publish(g.mx_activation_gradient("silu", held, x))
    four = g.mx_quantize(x, "mx4")
    w = g.mx_feed("mx4", (40, 100))
    g.publish(g.mx_linear(four, w, g.feed(BF16, (40,)), "relu", BF16))
    g.publish(g.mx_restore(four, F16))
    plan = native.describe(g.build())
    for line in ["mx_quantize bits=8 m=100 n=100", "mx_weight_gradient k=100 m=100 n=40", "mx_activation_gradient act=SILU m=100 n=100",
                 "mx_quantize bits=4 m=100 n=100", "mx_linear k=128 bias act=RELU m=100 n=40", "mx_restore bits=4 m=100 n=100"]:
        assert line in plan, plan


def status(builder):
    try:
        native.describe(builder.build())
    except native.NativeFailure as failure:
        return failure.status
    return 0


REFUSALS = {
    "quantize an integer tensor": (13, lambda g: g.publish(g.mx_quantize(g.feed(I32, (4, 32)), "mx4").codes)),
    "quantize a scalar": (8, lambda g: raw(g, "MX_QUANTIZE", [g.feed(F32, ())], [(U8, (16,)), (U8, (4,))], [4])),
    "quantize rank 5": (8, lambda g: g.publish(g.mx_quantize(g.feed(F32, (1, 1, 1, 1, 32)), "mx4").codes)),
    "quantize an empty last axis": (8, lambda g: raw(g, "MX_QUANTIZE", [g.feed(F32, (4, 0))], [(U8, (4, 0)), (U8, (4, 0))], [4])),
    "quantize to 5 bits": (13, lambda g: raw(g, "MX_QUANTIZE", [g.feed(F32, (4, 32))], [(U8, (4, 20)), (U8, (4, 4))], [5])),
    "codes of the wrong width": (9, lambda g: raw(g, "MX_QUANTIZE", [g.feed(F32, (4, 32))], [(U8, (4, 32)), (U8, (4, 4))], [4])),
    "scales of the wrong width": (9, lambda g: raw(g, "MX_QUANTIZE", [g.feed(F32, (4, 32))], [(U8, (4, 16)), (U8, (4, 1))], [4])),
    "one output": (9, lambda g: raw(g, "MX_QUANTIZE", [g.feed(F32, (4, 32))], [(U8, (4, 16))], [4])),
    "restore to integers": (13, lambda g: raw(g, "MX_RESTORE", held(g, "mx4", (4, 32)), [(I32, (4, 32))], [4, 32])),
    "restore to another width": (9, lambda g: raw(g, "MX_RESTORE", held(g, "mx4", (4, 32)), [(F32, (4, 33))], [4, 33])),
    "restore floats": (13, lambda g: raw(g, "MX_RESTORE", [g.feed(F32, (4, 16)), g.feed(U8, (4, 4))], [(F32, (4, 32))], [4, 32])),
    "strided codes": (8, lambda g: raw(g, "MX_RESTORE", [g.feed(U8, (4, 16), (32, 1)), g.feed(U8, (4, 4))], [(F32, (4, 32))], [4, 32])),
    "linear with 8-bit weights": (9, lambda g: raw(g, "MX_LINEAR", held(g, "mx4", (4, 32)) + held(g, "mx8", (8, 32)), [(F32, (4, 8))], [0])),
    "linear with other blocks": (9, lambda g: raw(g, "MX_LINEAR", held(g, "mx4", (4, 32)) + held(g, "mx4", (8, 64)), [(F32, (4, 8))], [0])),
    "linear with a batched weight": (8, lambda g: raw(g, "MX_LINEAR", held(g, "mx4", (4, 32)) + held(g, "mx4", (1, 8, 32)), [(F32, (4, 8))], [0])),
    "linear onto no columns": (8, lambda g: raw(g, "MX_LINEAR", held(g, "mx4", (4, 32)) + held(g, "mx4", (0, 32)), [(F32, (4, 0))], [0])),
    "linear with a bias of another type": (9, lambda g: raw(g, "MX_LINEAR", held(g, "mx4", (4, 32)) + held(g, "mx4", (8, 32)) + [g.feed(F32, (8,))], [(BF16, (4, 8))], [0])),
    "linear with a short bias": (9, lambda g: raw(g, "MX_LINEAR", held(g, "mx4", (4, 32)) + held(g, "mx4", (8, 32)) + [g.feed(F32, (7,))], [(F32, (4, 8))], [0])),
    "linear with a strided bias": (8, lambda g: raw(g, "MX_LINEAR", held(g, "mx4", (4, 32)) + held(g, "mx4", (8, 32)) + [g.feed(F32, (8,), (2,))], [(F32, (4, 8))], [0])),
    "linear with EXP as activation": (13, lambda g: raw(g, "MX_LINEAR", held(g, "mx4", (4, 32)) + held(g, "mx4", (8, 32)), [(F32, (4, 8))], [11])),
    "weight gradient from 4 bits": (9, lambda g: raw(g, "MX_WEIGHT_GRADIENT", held(g, "mx4", (4, 32)) + [g.feed(F32, (4, 8))], [(F32, (8, 32))], [32])),
    "weight gradient in 16 bits": (13, lambda g: raw(g, "MX_WEIGHT_GRADIENT", held(g, "mx8", (4, 32)) + [g.feed(F32, (4, 8))], [(BF16, (8, 32))], [32])),
    "weight gradient of other rows": (9, lambda g: raw(g, "MX_WEIGHT_GRADIENT", held(g, "mx8", (4, 32)) + [g.feed(F32, (5, 8))], [(F32, (8, 32))], [32])),
    "weight gradient of a strided gradient": (8, lambda g: raw(g, "MX_WEIGHT_GRADIENT", held(g, "mx8", (4, 32)) + [g.feed(F32, (4, 8), (1, 4))], [(F32, (8, 32))], [32])),
    "activation gradient of another type": (13, lambda g: raw(g, "MX_ACTIVATION_GRADIENT", held(g, "mx8", (4, 32)) + [g.feed(F32, (4, 32))], [(BF16, (4, 32))], [10])),
    "activation gradient of none": (13, lambda g: raw(g, "MX_ACTIVATION_GRADIENT", held(g, "mx8", (4, 32)) + [g.feed(F32, (4, 32))], [(F32, (4, 32))], [0])),
    "arithmetic on codes": (13, lambda g: raw(g, "ADD", [g.feed(U8, (4,)), g.feed(U8, (4,))], [(U8, (4,))], [])),
    "scalar arithmetic on codes": (13, lambda g: raw(g, "SCALAR_MAX", [g.feed(U8, (4,))], [(U8, (4,))], [1])),
}


def held(g, fmt, shape):
    mx = g.mx_feed(fmt, shape)
    return [mx.codes, mx.scales]


def raw(g, op, inputs, outputs, attrs):
    """A node as it stands, without the builder's own checks."""
    outs = [g._value(dtype, shape) for dtype, shape in outputs]
    g.nodes.append(program._Node(program.OPS[op], [v.index for v in inputs], [v.index for v in outs], list(attrs)))
    g.publish(outs[0])


@pytest.mark.parametrize("name", REFUSALS)
def test_refusals(name):
    want, make = REFUSALS[name]
    g = GraphBuilder()
    make(g)
    assert status(g) == want


def test_codes_that_do_not_start_on_16_bytes_are_refused():
    g = GraphBuilder()
    mx = g.mx_feed("mx8", (4, 32))
    g.publish(g.mx_restore(mx, F32))
    image = bytearray(g.build())
    for offset, want in [(16, 0), (8, 8), (1, 8)]:
        struct.pack_into("<Q", image, 64 + 40 * mx.codes.index + 16, offset)
        try:
            native.describe(bytes(image))
            got = 0
        except native.NativeFailure as failure:
            got = failure.status
        assert got == want


def test_builder_refuses_what_does_not_fit():
    g = GraphBuilder()
    with pytest.raises(ValueError):
        g.mx_linear(g.mx_feed("mx8", (4, 32)), g.mx_feed("mx4", (8, 32)))
    with pytest.raises(ValueError):
        g.mx_linear(g.mx_feed("mx4", (4, 64)), g.mx_feed("mx4", (8, 32)))
    with pytest.raises(ValueError):
        g.mx_weight_gradient(g.mx_feed("mx4", (4, 32)), g.feed(F32, (4, 8)))
    with pytest.raises(ValueError):
        g.mx_activation_gradient("relu", g.mx_feed("mx8", (4, 32)), g.feed(F32, (4, 31)))


def test_model_graphs():
    plan = native.describe(program.mlp_mx_inference_graph([784, 256, 10], 32, arg_max=True).image)
    assert [line.split()[0] for line in plan.splitlines()] == ["mx_quantize", "mx_linear", "mx_quantize", "mx_linear", "arg_max"]
    assert "act=RELU" in plan.splitlines()[1] and "act=" not in plan.splitlines()[3]
    for activation, held in [("relu", 3), ("gelu", 5)]:       # every layer's input; for GELU the two pre-activations too
        graph = program.mlp_training_graph([784, 256, 256, 10], 64, activation=activation, checkpoints="mx8")
        plan = native.describe(graph.image)
        steps = [line.split()[0] for line in plan.splitlines()]
        assert steps.count("mx_quantize") == held and steps.count("mx_weight_gradient") == 3 and steps.count("mx_activation_gradient") == 2
        assert graph.publications == program.mlp_training_graph([784, 256, 256, 10], 64, activation=activation).publications
    with pytest.raises(ValueError):
        program.mlp_training_graph([4, 4], 4, checkpoints="mx4")
    with pytest.raises(ValueError):
        program.mlp_mx_inference_graph([4, 4], (2, 3), arg_max=True)


def weight_from(q, how):
    """A weight over the memory of the quantised tensor q, wholly or in part."""
    def build(g):
        fed = g.mx_feed("mx4", q.shape)
        view = {"contiguous": g.contiguous, "permute": lambda v: g.permute(v, (0, 1)), "expand": lambda v: g.expand(v, v.shape)}
        if how == "same":
            return q
        if how == "fed":
            return fed
        if how == "codes only":
            return program.MxValue("mx4", q.shape, g.contiguous(q.codes), fed.scales)
        if how == "scales only":
            return program.MxValue("mx4", q.shape, fed.codes, g.contiguous(q.scales))
        if how == "twice":
            return program.MxValue("mx4", q.shape, g.contiguous(g.permute(q.codes, (0, 1))), g.permute(g.contiguous(q.scales), (0, 1)))
        return program.MxValue("mx4", q.shape, view[how](q.codes), view[how](q.scales))
    return build


@pytest.mark.parametrize("how,overlaps", [("fed", True), ("same", False), ("contiguous", False), ("permute", False), ("expand", False), ("twice", False),
                                          ("codes only", False), ("scales only", False)])
def test_a_product_only_overlaps_the_quantisation_that_does_not_make_its_weight(how, overlaps):
    """The product reads its weight before the launch in front has ended: not where that launch writes the weight's memory."""
    g = GraphBuilder()
    x = g.feed(F32, (40, 96))
    shape = program.MxValue("mx4", (40, 96), None, None)
    if how == "fed":
        weight = weight_from(shape, how)(g)
        q = g.mx_quantize(x, "mx4")
    else:
        q = g.mx_quantize(x, "mx4")
        weight = weight_from(q, how)(g)
    g.publish(g.mx_linear(q, weight))
    plan = native.describe(g.build()).splitlines()
    assert [line.split()[0] for line in plan] == ["mx_quantize", "mx_linear"]
    assert ("overlaps_quantize" in plan[1]) == overlaps, plan


def test_a_product_does_not_overlap_what_is_not_its_quantisation():
    g = GraphBuilder()
    x, y = g.feed(F32, (40, 96)), g.feed(F32, (50, 96))
    q = g.mx_quantize(x, "mx4")
    w = g.mx_quantize(y, "mx4")             # the weight is made last
    g.publish(g.mx_linear(q, w))
    g.publish(g.mx_linear(w, q))            # behind a product, not behind its quantisation
    assert "overlaps_quantize" not in native.describe(g.build())


def test_gates_of_relu_checkpoints_stay_open():
    """What a ReLU passed on is its gate in the backward pass: it is held so that nothing positive becomes zero."""
    steps = lambda activation: [line for line in native.describe(program.mlp_training_graph([784, 256, 256, 10], 64, activation=activation, checkpoints="mx8").image).splitlines()       # noqa: E731
                                if line.startswith("mx_quantize")]
    assert ["keep_nonzero" in line for line in steps("relu")] == [False, True, True]       # the model's input is no gate
    assert not any("keep_nonzero" in line for line in steps("gelu"))


@pytest.mark.parametrize("attrs,want", [([8], 0), ([8, 0], 0), ([8, 1], 0), ([4, 1], 0), ([8, 2], 13), ([8, 1, 0], 9), ([], 9)])
def test_attributes_of_quantise(attrs, want):
    g = GraphBuilder()
    raw(g, "MX_QUANTIZE", [g.feed(F32, (4, 32))], [(U8, (4, 16 if attrs[:1] == [4] else 32)), (U8, (4, 4))], attrs)
    assert status(g) == want
