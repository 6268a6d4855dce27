"""Block-scaled tensors in the model path on a B200: a stack whose weights are held in 4 bits, and training whose
backward pass reads 8-bit checkpoints, against the 64-bit implementations of mx_reference."""
import numpy as np
import pytest

import mx_reference as ref
from synaptik_b200 import native, nn, program

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = native.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("dims,batch,activation", [([32, 128, 1], 1, "relu"), ([784, 256, 256, 10], 33, "relu"), ([100, 300, 70], 200, "gelu_tanh"),
                                                   ([784, 512, 10], 700, "silu")])
def test_model_with_4_bit_weights(ctx, dims, batch, activation):
    """Layer by layer from the device's own layer inputs (prefixes of the stack), since quantisation steps a little
    difference up: what a layer makes of its input is held to the bound of one product (see test_gpu_mx)."""
    model = nn.Model(dims, ctx, seed=3, dtype="mx4", activation=activation)
    rng = np.random.default_rng(5)
    params = [rng.standard_normal(s).astype(np.float32) * (0.2 if len(s) == 1 else 1 / np.sqrt(s[1])) for s in model.param_shapes]
    model.load_parameters(params)
    held = model.parameters()
    for given, kept in zip(params, held):
        if given.ndim == 2:
            assert np.array_equal(kept, ref.values(*ref.quantize(given, "mx4"), "mx4", given.shape[1]).astype(np.float32))
    x = rng.standard_normal((batch, dims[0])).astype(np.float32)
    inputs = program.from_storage("bf16", program.to_storage("bf16", x)).astype(np.float64)
    for depth in range(1, len(dims)):
        part = nn.Model(dims[:depth + 1], ctx, dtype="mx4", activation=activation)
        part.load_parameters(params[:2 * depth])
        last = part.compute(x).astype(np.float64)          # the last layer of a stack has no activation
        w, b = held[2 * depth - 2].astype(np.float64), held[2 * depth - 1].astype(np.float64)
        a = ref.values(*ref.quantize(inputs, "mx4"), "mx4", dims[depth - 1])
        z, s = a @ w.T + b, np.abs(a) @ np.abs(w).T + np.abs(b)
        assert (np.abs(last - z) <= (dims[depth - 1] / 32 + 4) * 2.0 ** -23 * s + 2.0 ** -8 * 1.01 * np.abs(z)).all()
        part.close()
        # the device's own next input: this layer with its activation
        g = program.GraphBuilder()
        xm, wm, bm = g.feed(program.BF16, inputs.shape), g.mx_feed("mx4", w.shape), g.feed(program.BF16, b.shape)
        g.publish(g.mx_linear(g.mx_quantize(xm, "mx4"), wm, bm, activation, program.BF16))
        codes, scales = ref.quantize(params[2 * depth - 2], "mx4")
        got, = ref.helpers.run_image(ctx, g, [program.to_storage("bf16", inputs), codes, scales, program.to_storage("bf16", params[2 * depth - 1])])
        inputs = ref.read("bf16", got)
    logits, best = model.compute(x, arg_max=True)
    assert np.array_equal(logits, model.compute(x)) and np.array_equal(best, logits.argmax(1))
    with pytest.raises(ValueError):
        model.configure_training("mse", nn.Sgd(0.01))
    model.close()


def test_4_bit_model_over_leading_dimensions(ctx):
    model = nn.Model([64, 96, 32], ctx, seed=1, dtype="mx4")
    x = np.random.default_rng(0).standard_normal((3, 5, 64)).astype(np.float32)
    assert np.array_equal(model.compute(x), model.compute(x.reshape(15, 64)).reshape(3, 5, 32))
    model.close()


def reference_step(x, target, params, loss, activation):
    """Loss and gradients in 64 bits, the backward pass reading checkpoints of the forward pass's values."""
    layers = len(params) // 2
    a, inputs, zs = x.astype(np.float64), [], []
    for l in range(layers):
        inputs.append(a)
        z = a @ params[2 * l].astype(np.float64).T + params[2 * l + 1].astype(np.float64)
        zs.append(z)
        a = ref.activate(activation, z) if l + 1 < layers else z
    rows = x.shape[0]
    if loss == "mse":
        value, dz = ((a - target) ** 2).mean(), 2 * (a - target) / a.size
    else:
        e = np.exp(a - a.max(1, keepdims=True))
        p = e / e.sum(1, keepdims=True)
        value = -np.log(p[np.arange(rows), target]).mean()
        dz = p.copy()
        dz[np.arange(rows), target] -= 1
        dz /= rows
    grads = [None] * len(params)
    for l in range(layers - 1, -1, -1):
        grads[2 * l] = dz.T @ ref.values(*ref.quantize(inputs[l].astype(np.float32), "mx8"), "mx8", inputs[l].shape[1])
        grads[2 * l + 1] = dz.sum(0)
        if l:
            kept = inputs[l] if activation == "relu" else zs[l - 1]
            kept = ref.values(*ref.quantize(kept.astype(np.float32), "mx8"), "mx8", kept.shape[1])
            dz = (dz @ params[2 * l].astype(np.float64)) * ref.slope(activation, kept)
    return value, grads


@pytest.mark.parametrize("dims,batch,loss,activation", [([32, 128, 1], 1024, "mse", "relu"), ([784, 256, 256, 10], 300, "ce", "relu"),
                                                        ([60, 130, 70, 5], 77, "ce", "gelu"), ([64, 64, 3], 1, "mse", "tanh")])
def test_training_from_8_bit_checkpoints(ctx, dims, batch, loss, activation):
    """Gradients against the 64-bit step with the same checkpoints.  An element of a checkpoint may round the other way
    where the FLOAT32 value differs from the 64-bit one next to a tie: one step of 2^-3 in one of many terms, with
    probability 2^-24 * sqrt(K) / 2^-4; 2e-3 of the norm allows for a few hundred of them."""
    model = nn.Model(dims, ctx, seed=2, activation=activation, checkpoints="mx8")
    plain = nn.Model(dims, ctx, seed=2, activation=activation)
    rng = np.random.default_rng(8)
    x = rng.standard_normal((batch, dims[0])).astype(np.float32)
    target = rng.integers(0, dims[-1], batch) if loss == "ce" else rng.standard_normal((batch, dims[-1])).astype(np.float32)
    for m in (model, plain):
        m.configure_training(loss, nn.Sgd(0.01))
    value, grads = model.gradients(x, target)
    plain_value, plain_grads = plain.gradients(x, target)
    want_value, want = reference_step(x, target, model.parameters(), loss, activation)
    assert value == plain_value                        # the forward pass does not change
    assert abs(value - want_value) <= 1e-5 * abs(want_value)
    for got, exact, other in zip(grads, want, plain_grads):
        assert np.linalg.norm(got - exact) <= 2e-3 * np.linalg.norm(exact) + 1e-12
        # against FLOAT32 checkpoints: each held value is off by at most 2^-4 of itself, each slope likewise
        assert np.linalg.norm(got - other) <= 0.25 * np.linalg.norm(other) + 1e-12
    before = model.parameters()
    model.train(x, target)
    for p, q, g in zip(before, model.parameters(), grads):
        assert np.allclose(q, p - np.float32(0.01) * g, rtol=1e-6, atol=1e-7)
    # the same step again gives the same bits
    model.load_parameters(before)
    again = model.gradients(x, target)
    assert again[0] == value and all(np.array_equal(a, b) for a, b in zip(again[1], grads))
    model.close()
    plain.close()


def test_non_finite_inputs_refuse_the_step(ctx):
    """A NaN among the inputs makes NaN gradients from its checkpoint, and the optimizer leaves everything as it was."""
    model = nn.Model([64, 64, 4], ctx, seed=2, checkpoints="mx8")
    model.configure_training("mse", nn.Sgd(0.01))
    x = np.ones((8, 64), dtype=np.float32)
    x[3, 7] = np.nan
    before = model.parameters()
    with pytest.raises(native.NativeFailure):
        model.train(x, np.zeros((8, 4), dtype=np.float32))
    assert all(np.array_equal(a, b) for a, b in zip(before, model.parameters()))
    model.close()


def test_two_executables_share_buffers_and_contexts_do_not_mix(ctx):
    """Two programs on the same buffers, run in turn and twice each, and the same on another context of the device."""
    rng = np.random.default_rng(1)
    other = native.Context(0)
    results = []
    for c in (ctx, other):
        x = rng.standard_normal((300, 160)).astype(np.float32) if not results else x
        w = rng.standard_normal((520, 160)).astype(np.float32) if not results else w
        g = program.GraphBuilder()
        xv = g.feed(program.F32, x.shape)
        wv = g.feed(program.F32, w.shape)
        g.publish(g.mx_linear(g.mx_quantize(xv, "mx4"), g.mx_quantize(wv, "mx4")))
        first, second = native.Executable(c, g.build()), native.Executable(c, g.build())
        buffers = [c.upload(x), c.upload(w)]
        outs = [c.buffer(300 * 520 * 4) for _ in range(2)]
        for _ in range(2):
            first.enqueue(buffers, [outs[0]])
            second.enqueue(buffers, [outs[1]])
        first.finish()
        second.finish()
        results += [o.download(np.float32, (300, 520)) for o in outs]
        first.close()
        second.close()
        for b in buffers + outs:
            b.close()
    other.close()
    assert all(np.array_equal(results[0], r) for r in results[1:])
    xv, wv = (ref.values(*ref.quantize(a, "mx4"), "mx4", 160) for a in (x, w))
    assert (np.abs(results[0] - xv @ wv.T) <= 9 * 2.0 ** -23 * (np.abs(xv) @ np.abs(wv).T)).all()


def test_one_tensor_as_both_operands(ctx):
    """x . x^T: the quantised tensor serves as input and as weight of one product."""
    for rows in (40, 2000):
        x = np.random.default_rng(rows).standard_normal((rows, 96)).astype(np.float32)
        g = program.GraphBuilder()
        held = g.mx_quantize(g.feed(program.F32, x.shape), "mx4")
        g.publish(g.mx_linear(held, held))
        got, = ref.helpers.run_image(ctx, g, [x])
        v = ref.values(*ref.quantize(x, "mx4"), "mx4", 96)
        assert (np.abs(got - v @ v.T) <= 7 * 2.0 ** -23 * (np.abs(v) @ np.abs(v).T)).all()


def test_checkpoints_take_less_memory(ctx):
    """A training program with 8-bit checkpoints reuses the memory of what its backward pass no longer reads."""
    torch = pytest.importorskip("torch")
    dims, batch = [256, 1024, 1024, 1024, 1024, 16], 8192
    used, grads = {}, {}
    rng = np.random.default_rng(0)
    x, target = rng.standard_normal((batch, dims[0])).astype(np.float32), rng.integers(0, dims[-1], batch)
    for kind in (None, "mx8"):
        model = nn.Model(dims, ctx, seed=4, checkpoints=kind)
        model.configure_training("ce", nn.Sgd(0.01))
        ctx.synchronize()
        free = torch.cuda.mem_get_info(0)[0]
        model.training_state(batch)
        used[kind] = free - torch.cuda.mem_get_info(0)[0]
        grads[kind] = model.gradients(x, target)
        model.close()
    assert used["mx8"] < 0.7 * used[None], used
    assert grads["mx8"][0] == grads[None][0]
    for a, b in zip(grads["mx8"][1], grads[None][1]):
        assert np.linalg.norm(a - b) <= 0.25 * np.linalg.norm(b)


def test_two_threads_with_a_context_each(ctx):
    """Programs of both tensor-core products run from two threads at once, each on its own context."""
    import threading
    rng = np.random.default_rng(3)
    x = rng.standard_normal((700, 320)).astype(np.float32)
    w = rng.standard_normal((1100, 320)).astype(np.float32)
    up = rng.standard_normal((700, 600)).astype(np.float32)
    results, failures = {}, []

    def work(name):
        try:
            c = native.Context(0)
            got = []
            for _ in range(5):
                g = program.GraphBuilder()
                xv, wv, uv = g.feed(program.F32, x.shape), g.feed(program.F32, w.shape), g.feed(program.F32, up.shape)
                g.publish(g.mx_linear(g.mx_quantize(xv, "mx4"), g.mx_quantize(wv, "mx4")))
                g.publish(g.mx_weight_gradient(g.mx_quantize(xv, "mx8"), uv))
                got.append(ref.helpers.run_image(c, g, [x, w, up]))
            c.close()
            results[name] = got
        except Exception as e:      # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures
    first = results[0][0]
    for got in results[0] + results[1]:
        assert all(np.array_equal(a, b) for a, b in zip(first, got))


def test_small_activations_beside_large_ones_keep_their_gradient(ctx):
    """One unit at 1000 and others at 1e-6 to 1e-3 in a block: each open unit's gradient is what FLOAT32 checkpoints give it
    (the inputs are exact in 8 bits), each closed unit's is zero."""
    hidden = 64
    target = np.zeros((4, 1), dtype=np.float32)
    x = np.ones((4, 2), dtype=np.float32)
    w0 = np.zeros((hidden, 2), dtype=np.float32)
    w0[:, 0] = np.where(np.arange(hidden) % 3 == 0, -1, 1) * np.geomspace(1e-6, 1e-3, hidden)
    w0[0, 0] = w0[33, 0] = 1000
    w1 = np.linspace(0.5, 1.5, hidden, dtype=np.float32)[None]
    grads = []
    for kind in (None, "mx8"):
        model = nn.Model([2, hidden, 1], ctx, checkpoints=kind)
        model.load_parameters([w0, np.zeros(hidden, np.float32), w1, np.zeros(1, np.float32)])
        model.configure_training("mse", nn.Sgd(0.01))
        grads.append(model.gradients(x, target)[1])
        model.close()
    opened = w0[:, 0] > 0
    assert (grads[1][0][opened] != 0).all() and (grads[1][0][~opened] == 0).all()
    # four equal rows: each result is a sum of at most 12 exact products, one rounding each
    assert np.allclose(grads[1][0], grads[0][0], rtol=16 * 2.0 ** -23, atol=0)
    assert np.allclose(grads[1][1], grads[0][1], rtol=16 * 2.0 ** -23, atol=0)


@pytest.mark.parametrize("dims,batch,activation", [([256, 512, 512, 512, 16], 2048, "relu"), ([100, 300, 260, 10], 700, "gelu"), ([64, 384, 384, 384, 384, 8], 1024, "tanh")])
def test_shared_memory_does_not_change_a_bit(ctx, dims, batch, activation):
    """Intermediates of a program with 8-bit checkpoints share memory.  Published ones have memory of their own, and who writes
    the operand planes of a product changes which of them live when: the gradients are the same bits."""
    rng = np.random.default_rng(batch)
    x, target = rng.standard_normal((batch, dims[0])).astype(np.float32), rng.integers(0, dims[-1], batch).astype(np.int32)
    params = [(rng.standard_normal(s) / np.sqrt(s[-1])).astype(np.float32) for l in range(len(dims) - 1) for s in ((dims[l + 1], dims[l]), (dims[l + 1],))]
    results = []
    try:
        for publish in (False, True):
            for fused in (1, 0, 2, 3):
                for timed in (0, 1):
                    ctx.set_option("fused_planes", fused)
                    ctx.set_option("time_steps", timed)
                    graph = program.mlp_training_graph(dims, batch, "ce", activation=activation, publish_activations=publish, checkpoints="mx8")
                    exe = native.Executable(ctx, graph.image)
                    feeds = [ctx.upload(a) for a in [x, target, np.ones(1, np.float32)] + params]
                    outs = [ctx.buffer(max(int(np.prod(graph.shapes[name])) * 4, 4)) for name in graph.publications]
                    for _ in range(2):
                        exe.enqueue(feeds, outs)
                    exe.finish()
                    got = {name: b.download(np.float32, graph.shapes[name]) for name, b in zip(graph.publications, outs)}
                    results.append({name: v for name, v in got.items() if name in graph.publications[:1 + len(params)]})
                    exe.close()
                    for b in feeds + outs:
                        b.close()
    finally:
        ctx.set_option("fused_planes", 1)
        ctx.set_option("time_steps", 0)
    assert len(results[0]) == 1 + len(params)
    for other in results[1:]:
        assert other.keys() == results[0].keys()
        assert all(np.array_equal(other[name], results[0][name]) for name in other)


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("activation", ["relu", "tanh", "sigmoid", "silu", "gelu_tanh", "gelu"])
def test_checkpointed_training_of_every_activation(ctx, activation, bias):
    """Against FLOAT32 checkpoints: each held value is off by at most 2^-4 of itself, each slope likewise."""
    dims, batch = [33, 96, 65, 7], 130
    rng = np.random.default_rng(6)
    x, target = rng.standard_normal((batch, dims[0])).astype(np.float32), rng.standard_normal((batch, dims[-1])).astype(np.float32)
    grads = []
    for kind in (None, "mx8"):
        model = nn.Model(dims, ctx, seed=5, bias=bias, activation=activation, checkpoints=kind)
        model.configure_training("mse", nn.Sgd(0.01))
        grads.append(model.gradients(x, target))
        model.close()
    assert grads[0][0] == grads[1][0]
    for a, b in zip(grads[1][1], grads[0][1]):
        assert np.linalg.norm(a - b) <= 0.25 * np.linalg.norm(b)
