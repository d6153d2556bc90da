"""A cache of 8-bit integers in use: pages and slots, rotary positions with the quantising write,
attention of rows and of runs, reading back, between quantized projections, over steps in
which prompts join decoding requests.  Against 64 bits: the cache's elements, read back, lie within
2.5 steps of their block's scale of the projections' k and v (the header's bound, and the
projections' own 2^-20), and the outputs are those of attention over what the cache holds: q is
rounded to 16 bits once, so an output element, a sum over heads * dim attention values, is held to
2^-9 (fp16; bf16 2^-6) of the largest output, as for 16-bit caches."""
import numpy as np
import pytest

import attn_ref as ref
from attn_ref import BF16, F16, F32
from openmini_qmm import synth

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV, DIM, PAGE, MAX_PAGES, REQUESTS = 512, 8, 2, 64, 32, 6, 4


class Layer:
    def __init__(self, qmm, orc, seed, cache_t, q_t, block, shared=None, axes=1):
        shapes = [(HEADS * DIM, HIDDEN), (KV * DIM, HIDDEN), (KV * DIM, HIDDEN), (HIDDEN, HEADS * DIM)]
        blocks = [synth.weight_blocks(7, n, k, seed=seed + i, sigma=0.05) for i, (n, k) in enumerate(shapes)]
        self.w = [orc.dequantize(7, b, n * k).reshape(n, k).astype(np.float64) for b, (n, k) in zip(blocks, shapes)]
        self.weights = qmm.AttentionWeights(*[qmm.QuantizedWeight(7, b, n, k) for b, (n, k) in zip(blocks, shapes)])
        self.freq = qmm.rope_frequencies(DIM // 2)
        self.cache = qmm.KVCache.allocate(cache_t, 24, PAGE, KV, DIM, block=block) if cache_t == qmm.DType.I8 else \
            qmm.KVCache.allocate(cache_t, 24, PAGE, KV, DIM)
        self.step = qmm.CachedAttention(self.weights, qmm.Rope(self.freq), self.cache, HEADS, 128, q_t,
                                        attention=shared.step.attention if shared else None,
                                        prompt=shared.step.prompt if shared else qmm.PromptAttention(HEADS, KV, DIM, q_t, F32))


def _read(qmm, layer, tables, lens, stream):
    """Every request's keys and values, fp32."""
    starts = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    outs = [qmm.DeviceBuffer(int(starts[-1]) * KV * DIM * 4) for _ in range(2)]
    layer.cache.read(tables, MAX_PAGES, qmm.DeviceBuffer.from_numpy(starts), len(lens), int(starts[-1]), *outs, F32, stream=stream)
    both = [o.download(np.float32, (int(starts[-1]), KV, DIM), stream).astype(np.float64) for o in outs]
    return [tuple(b[starts[r]:starts[r + 1]] for b in both) for r in range(len(lens))]


@pytest.mark.parametrize("q_t", [F16, BF16])
@pytest.mark.parametrize("cache_t,block", [(4, 8), (4, 16), (4, 32), (None, 0)])
def test_prompts_and_decoding(qmm, orc, cache_t, block, q_t):
    i8 = cache_t == 4
    cache_t = qmm.DType.I8 if i8 else q_t
    rng = np.random.default_rng(30 + block)
    first = Layer(qmm, orc, 0xC00, cache_t, q_t, block)
    layers = [first, Layer(qmm, orc, 0xC10, cache_t, q_t, block, first)]
    plan = qmm.StepPlan(PAGE, REQUESTS, 128, MAX_PAGES)
    tables, head = qmm.DeviceBuffer(REQUESTS * MAX_PAGES * 4), 0
    tables.fill(0xFF)
    d_free = qmm.DeviceBuffer.from_numpy(rng.permutation(24).astype(np.int32))
    cached = np.zeros(REQUESTS, np.int32)
    exact = [[tuple(np.zeros((0, KV, DIM)) for _ in range(2)) for _ in range(REQUESTS)] for _ in layers]
    s = qmm.Stream()
    # two prompts; they decode while a third request's prompt comes in pieces and a fourth's whole;
    # all decode; a request that asks for more than its table is refused
    for new, decoding in (([40, 3, 0, 0], 0), ([1, 1, 33, 0], 2), ([1, 1, 5, 70], 2), ([1, 1, 1, 1], 4), ([1, 1, 1, 1], None), ([1, 1, 1, 125], 3)):
        tokens = min(sum(new), 128)
        print(f"step {new} on {cached.tolist()} decoding {decoding}", flush=True)
        plan.run(qmm.DeviceBuffer.from_numpy(cached), qmm.DeviceBuffer.from_numpy(np.array(new, np.int32)), REQUESTS, tables, d_free, 24,
                 d_head=qmm.DeviceBuffer.from_numpy(np.array([head], np.int32)), stream=s.handle)
        counts = plan.counts.download(np.int32, (4,), s.handle)
        lens = plan.lens.download(np.int32, (REQUESTS,), s.handle)
        head = int(counts[3])
        refused = [c + n > MAX_PAGES * PAGE for c, n in zip(cached, new)]
        assert counts[2] == sum(refused)
        rows = [r for r, n in enumerate(new) for _ in range(n)][:tokens]
        at = np.array([int(cached[r]) + j for r, n in enumerate(new) for j in range(n)][:tokens])
        x = rng.standard_normal((tokens, HIDDEN)).astype(np.float32)
        d_x = qmm.DeviceBuffer.from_numpy(x)
        for layer, memory in zip(layers, exact):
            d_out = qmm.DeviceBuffer(tokens * HIDDEN * 4)
            layer.step.forward_device(d_x, plan, tables, REQUESTS, tokens, d_out, stream=s.handle, decoding=decoding)
            got = d_out.download(np.float32, (tokens, HIDDEN), s.handle).astype(np.float64)
            q, k, v = (x.astype(np.float64) @ w.T for w in layer.w[:3])
            q = ref.decode(ref.encode(ref.rope(q.reshape(tokens, HEADS, DIM), at[None], layer.freq, [0] * (DIM // 2)), q_t), q_t)
            k, v = ref.rope(k.reshape(tokens, KV, DIM), at[None], layer.freq, [0] * (DIM // 2)), v.reshape(tokens, KV, DIM)
            for j, r in enumerate(rows):
                if not refused[r]:
                    memory[r] = tuple(np.concatenate([m, n[j:j + 1]]) for m, n in zip(memory[r], (k, v)))
            held = _read(qmm, layer, tables, lens, s.handle)
            for r in range(REQUESTS):
                for back, true in zip(held[r], memory[r]):
                    if not len(true):
                        continue
                    off = np.abs(back - true)
                    if i8:  # a block's largest element is at least a quarter under its scale's 127
                        most = np.array([np.abs(true[b // block * block:b // block * block + block]).max((0, 2)) for b in range(len(true))])
                        assert np.all(off <= (2.5 * 1.25 / 127 + 2.0 ** -10) * most[..., None]), (r, (off / most[..., None]).max())
                    else:
                        assert np.all(off <= 2 * ref.ROUND[q_t] * np.abs(true) + 2.0 ** -18 * np.abs(true).max()), r
            want = np.zeros((tokens, HEADS * DIM))
            for j, r in enumerate(rows):
                if not refused[r]:
                    want[j] = ref.attention(q[j], *(a[:at[j] + 1] for a in held[r]), DIM ** -0.5)[0].ravel()
            want = want @ layer.w[3].T
            off = np.abs(got - want).max() / np.abs(want).max()
            assert off <= (2.0 ** -9 if q_t == F16 else 2.0 ** -6), off
            for j, r in enumerate(rows):
                assert not refused[r] or not got[j].any()
        cached = lens


def test_refusals(qmm, orc):
    layer = Layer(qmm, orc, 0x1300, qmm.DType.I8, F16, 16)
    plan, d = qmm.StepPlan(PAGE, 2, 64, MAX_PAGES), qmm.DeviceBuffer(1 << 18)
    for requests, tokens, decoding in ((2, 5, 3), (2, 1, 2), (2, 5, 2), (2, 5, -1)):
        with pytest.raises(qmm.InvalidInput, match="decoding requests"):
            layer.step.forward_device(d, plan, d, requests, tokens, d, decoding=decoding)
    with pytest.raises(qmm.InvalidInput, match="shared attention has heads"):
        layer.step.prompt = qmm.PromptAttention(HEADS * 2, KV, DIM, F16, F32)
    with pytest.raises(qmm.InvalidInput, match="other types"):
        layer.step.prompt = qmm.PromptAttention(HEADS, KV, DIM, F16)
    layer.step.prompt = qmm.PromptAttention(HEADS, KV, DIM, F16, F32, window=7)
    with pytest.raises(qmm.InvalidInput, match="window"):
        layer.step.forward_device(d, plan, d, 2, 5, d, decoding=1)
    layer.step.prompt = None
    with pytest.raises(qmm.InvalidInput, match="runs need"):
        layer.step.forward_device(d, plan, d, 2, 5, d, decoding=1)
