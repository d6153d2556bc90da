"""CachedAttention in its default type, and on both sides of the rows from which the framework's
host calls take the prefill GEMM.  q, k and v are rounded to bf16 once (2^-8); an output element is
held to 2^-6 of the largest output, twice the two roundings that an attention value passes, and
the projections' own 2^-20."""
import numpy as np
import pytest

import attn_ref as ref
from attn_ref import BF16
from openmini_qmm import synth

pytestmark = pytest.mark.gpu
HIDDEN, HEADS, KV, DIM, PAGE = 512, 8, 2, 64, 16


def _round(x):
    return ref.decode(ref.encode(x, BF16), BF16)


@pytest.mark.parametrize("new", [[40, 1, 0, 20], [1, 1, 1, 1], [90, 60, 1, 3], [200, 0, 0, 1]])
def test_prompts_and_decoding_rows(qmm, orc, new):
    """Requests that hold 0, 37, 5 and 200 tokens already (a step of their own)."""
    shapes = [(HEADS * DIM, HIDDEN), (KV * DIM, HIDDEN), (KV * DIM, HIDDEN), (HIDDEN, HEADS * DIM)]
    blocks = [synth.weight_blocks(7, n, k, seed=0x1300 + i, sigma=0.05) for i, (n, k) in enumerate(shapes)]
    w = [orc.dequantize(7, b, n * k).reshape(n, k).astype(np.float64) for b, (n, k) in zip(blocks, shapes)]
    weights = qmm.AttentionWeights(*[qmm.QuantizedWeight(7, b, n, k) for b, (n, k) in zip(blocks, shapes)])
    freq = qmm.rope_frequencies(DIM // 2)
    cache = qmm.KVCache.allocate(BF16, 64, PAGE, KV, DIM)
    step = qmm.CachedAttention(weights, qmm.Rope(freq), cache, HEADS, 256)
    plan, tables = qmm.StepPlan(PAGE, 4, 256, 32), qmm.DeviceBuffer(4 * 32 * 4)
    buf, rng = qmm.DeviceBuffer.from_numpy, np.random.default_rng(sum(new))
    free = buf(rng.permutation(64).astype(np.int32))
    cached, head = np.zeros(4, np.int32), 0
    memory = [(np.zeros((0, KV, DIM)),) * 2 for _ in range(4)]
    for n in ([0, 37, 5, 200], new):
        tokens = sum(n)
        print(f"bf16 step {n} on {cached.tolist()}", flush=True)
        plan.run(buf(cached), buf(np.array(n, np.int32)), 4, tables, free, 64, d_head=buf(np.array([head], np.int32)))
        rows = [r for r, k in enumerate(n) for _ in range(k)]
        pos = np.array([[int(cached[r]) + j for r, k in enumerate(n) for j in range(k)]])
        x = rng.standard_normal((tokens, HIDDEN)).astype(np.float32)
        d_out = qmm.DeviceBuffer(tokens * HIDDEN * 4)
        step.forward_device(buf(x), plan, tables, 4, tokens, d_out)
        got = d_out.download(np.float32, (tokens, HIDDEN)).astype(np.float64)
        q, k, v = (x.astype(np.float64) @ m.T for m in w[:3])
        q = _round(ref.rope(q.reshape(tokens, HEADS, DIM), pos, freq, [0] * 32))
        k, v = _round(ref.rope(k.reshape(tokens, KV, DIM), pos, freq, [0] * 32)), _round(v.reshape(tokens, KV, DIM))
        want = np.zeros((tokens, HEADS * DIM))
        for j, r in enumerate(rows):
            memory[r] = tuple(np.concatenate([m, t[j:j + 1]]) for m, t in zip(memory[r], (k, v)))
            want[j] = ref.attention(q[j], *memory[r], DIM ** -0.5)[0].ravel()
        want = want @ w[3].T
        assert np.max(np.abs(got - want)) <= 2.0 ** -6 * np.max(np.abs(want)), float(np.max(np.abs(got - want)) / np.max(np.abs(want)))
        counts = plan.counts.download(np.int32, (4,))
        head, cached = int(counts[3]), plan.lens.download(np.int32, (4,))
        assert counts[0] == tokens and counts[2] == 0
