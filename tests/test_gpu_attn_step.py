"""The attention step in use: CachedAttention between quantized projections, prompts and
decoding requests together, against 64 bits.  q, k and v are rounded to fp16 once (2^-11),
so an output element, a sum over heads * dim attention values, is held to 2^-9 of the
largest output: twice the two roundings that an attention value passes, and the projections'
own 2^-20."""
import numpy as np
import pytest

import attn_ref as ref
from attn_ref import BF16, F16, F8
from openmini_qmm import synth

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV, DIM, PAGE, MAX_PAGES = 512, 8, 2, 64, 16, 6


class Layer:
    def __init__(self, qmm, orc, seed, cache_t, axes):
        shapes = [(HEADS * DIM, HIDDEN), (KV * DIM, HIDDEN), (KV * DIM, HIDDEN), (HIDDEN, HEADS * DIM)]
        blocks = [synth.weight_blocks(7, n, k, seed=seed + i, sigma=0.05) for i, (n, k) in enumerate(shapes)]
        self.w = [orc.dequantize(7, b, n * k).reshape(n, k).astype(np.float64) for b, (n, k) in zip(blocks, shapes)]
        self.weights = qmm.AttentionWeights(*[qmm.QuantizedWeight(7, b, n, k) for b, (n, k) in zip(blocks, shapes)])
        self.freq = qmm.rope_frequencies(DIM // 2)
        self.axis = qmm.rope_axes([DIM // 2] if axes == 1 else [8, 12, 12], "cycled" if axes > 1 else "blocks")
        self.cache = qmm.KVCache.allocate(cache_t, 24, PAGE, KV, DIM, k_scale=0.01 if cache_t == F8 else 1.0,
                                          v_scale=0.01 if cache_t == F8 else 1.0)
        self.step = qmm.CachedAttention(self.weights, qmm.Rope(self.freq, axes=self.axis, n_axes=axes), self.cache, HEADS, 64, F16)


def _round(x, t, scale=1.0):
    return ref.decode(ref.encode(x / scale, t), t) * scale


@pytest.mark.parametrize("cache_t,axes", [(F16, 1), (F16, 3)])
def test_prompts_and_decoding(qmm, orc, cache_t, axes):
    rng = np.random.default_rng(30 + axes)
    layers = [Layer(qmm, orc, 0xC00 + 16 * i, cache_t, axes) for i in range(2)]
    layers[1].step.attention = layers[0].step.attention  # one workspace for layers that follow each other
    plan = qmm.StepPlan(PAGE, 3, 64, MAX_PAGES)
    tables, head = qmm.DeviceBuffer(3 * MAX_PAGES * 4), 0
    tables.fill(0xFF)
    free = rng.permutation(24).astype(np.int32)
    d_free = qmm.DeviceBuffer.from_numpy(free)
    cached = np.zeros(3, np.int32)
    seen = [[(np.zeros((0, KV, DIM)),) * 2 for _ in range(3)] for _ in layers]
    s = qmm.Stream()
    # a prompt of 5 and one of 17; the third request's prompt while the others decode; a step
    # that one sits out; a full step
    for new in ([5, 17, 0], [1, 1, 33], [1, 0, 1], [1, 1, 1], [1, 1, 1]):
        tokens = sum(new)
        print(f"step {new} on {cached.tolist()}", flush=True)
        d_head = qmm.DeviceBuffer.from_numpy(np.array([head], np.int32))
        plan.run(qmm.DeviceBuffer.from_numpy(cached), qmm.DeviceBuffer.from_numpy(np.array(new, np.int32)), 3, tables, d_free, 24,
                 d_head=d_head, stream=s.handle)
        rows = [r for r, n in enumerate(new) for _ in range(n)]
        at = [int(cached[r]) + j for r, n in enumerate(new) for j in range(n)]
        pos = np.array([at] if axes == 1 else [at, [p % 7 for p in at], [p % 5 for p in at]], np.int32)
        d_pos = None if axes == 1 else qmm.DeviceBuffer.from_numpy(pos)
        x = rng.standard_normal((tokens, HIDDEN)).astype(np.float32)
        d_x = qmm.DeviceBuffer.from_numpy(x)
        for layer, memory in zip(layers, seen):
            d_out = qmm.DeviceBuffer(tokens * HIDDEN * 4)
            layer.step.forward_device(d_x, plan, tables, 3, tokens, d_out, d_positions=d_pos, stream=s.handle)
            got = d_out.download(np.float32, (tokens, HIDDEN), s.handle).astype(np.float64)
            x64 = x.astype(np.float64)
            q, k, v = (x64 @ w.T for w in layer.w[:3])
            q = _round(ref.rope(q.reshape(tokens, HEADS, DIM), pos, layer.freq, layer.axis), F16)
            k = _round(ref.rope(k.reshape(tokens, KV, DIM), pos, layer.freq, layer.axis), cache_t)
            v = _round(v.reshape(tokens, KV, DIM), cache_t)
            want = np.zeros((tokens, HEADS * DIM))
            for j, r in enumerate(rows):
                memory[r] = tuple(np.concatenate([m, n[j:j + 1]]) for m, n in zip(memory[r], (k, v)))
                want[j] = ref.attention(q[j], *memory[r], DIM ** -0.5)[0].ravel()
            want = want @ layer.w[3].T
            assert np.max(np.abs(got - want)) <= 2.0 ** -9 * np.max(np.abs(want)), float(np.max(np.abs(got - want)) / np.max(np.abs(want)))
        counts = plan.counts.download(np.int32, (4,), s.handle)
        assert counts[0] == tokens and counts[2] == 0
        head = int(counts[3])
        cached = plan.lens.download(np.int32, (3,), s.handle)


def test_e4m3_cache_runs(qmm, orc):
    """The same with an e4m3 cache: its 4-bit mantissas leave about 2^-4 / sqrt(keys) of an
    attention value; held to a quarter of the largest output."""
    layer = Layer(qmm, orc, 0xD00, F8, 1)
    plan, tables = qmm.StepPlan(PAGE, 1, 64, MAX_PAGES), qmm.DeviceBuffer(MAX_PAGES * 4)
    free = qmm.DeviceBuffer.from_numpy(np.arange(24, dtype=np.int32))
    x = np.random.default_rng(9).standard_normal((40, HIDDEN)).astype(np.float32)
    buf = qmm.DeviceBuffer.from_numpy
    plan.run(buf(np.zeros(1, np.int32)), buf(np.array([40], np.int32)), 1, tables, free, 24)
    d_out = qmm.DeviceBuffer(40 * HIDDEN * 4)
    print("step on an e4m3 cache", flush=True)
    layer.step.forward_device(buf(x), plan, tables, 1, 40, d_out)
    got = d_out.download(np.float32, (40, HIDDEN)).astype(np.float64)
    q, k, v = (x.astype(np.float64) @ w.T for w in layer.w[:3])
    pos = np.arange(40)[None]
    q, k = (ref.rope(t.reshape(40, -1, DIM), pos, layer.freq, layer.axis) for t in (q, k))
    v = v.reshape(40, KV, DIM)
    want = np.stack([ref.attention(q[j], k[:j + 1], v[:j + 1], DIM ** -0.5)[0].ravel() for j in range(40)]) @ layer.w[3].T
    assert np.max(np.abs(got - want)) <= 0.25 * np.max(np.abs(want))


def test_refusals(qmm, orc):
    layer = Layer(qmm, orc, 0xE00, F16, 1)
    rope = qmm.Rope(layer.freq)
    with pytest.raises(qmm.InvalidInput, match="query"):
        qmm.CachedAttention(layer.weights, rope, layer.cache, HEADS * 2, 8, F16)
    with pytest.raises(qmm.InvalidInput, match="other types"):
        qmm.CachedAttention(layer.weights, rope, layer.cache, HEADS, 8, F16, attention=qmm.PagedAttention(HEADS, KV, DIM, BF16))
    w = layer.weights
    with pytest.raises(qmm.InvalidInput, match="no o_proj"):
        qmm.CachedAttention(qmm.AttentionWeights(w.q_proj, w.k_proj, w.v_proj), rope, layer.cache, HEADS, 8, F16)
    plan = qmm.StepPlan(PAGE, 1, 64, MAX_PAGES)
    d = qmm.DeviceBuffer(1 << 18)
    with pytest.raises(qmm.InvalidInput, match="planned for"):
        layer.step.forward_device(d, plan, d, 1, 65, d)
    with pytest.raises(qmm.InvalidInput):
        qmm.StepPlan(PAGE, 1, 8, 4, buffers={"slot": d})
    with pytest.raises(qmm.InvalidInput):
        plan.run(d, d, 2, d, d, 4)


def test_max_pages(qmm, orc):
    """Fewer columns of the same tables, as many as the step needs: the same outputs, to
    2^-16 of the largest: fp32 sums of the same products in other orders, then a sum of 512."""
    layer = Layer(qmm, orc, 0xF00, F16, 1)
    width, buf = 400, qmm.DeviceBuffer.from_numpy
    plan, tables = qmm.StepPlan(PAGE, 2, 64, width), qmm.DeviceBuffer(2 * width * 4)
    plan.run(buf(np.zeros(2, np.int32)), buf(np.array([20, 33], np.int32)), 2, tables, buf(np.arange(24, dtype=np.int32)), 24)
    d_x, outs = buf(np.random.default_rng(10).standard_normal((53, HIDDEN)).astype(np.float32)), []
    for max_pages in (None, 3):
        d_out = qmm.DeviceBuffer(53 * HIDDEN * 4)
        layer.step.forward_device(d_x, plan, tables, 2, 53, d_out, max_pages=max_pages)
        outs.append(d_out.download(np.float32, (53, HIDDEN)))
    assert np.max(np.abs(outs[0] - outs[1])) <= 2.0 ** -16 * np.max(np.abs(outs[0]))
    for bad in (0, width + 1):
        with pytest.raises(qmm.InvalidInput, match="max_pages"):
            layer.step.forward_device(d_x, plan, tables, 2, 53, d_out, max_pages=bad)
