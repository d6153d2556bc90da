"""The projections of one transformer layer on quantized weights.

Mirrors the two places where src/model/inference/model.rs (openmini-server/) runs
several linear layers on one input:
  * FFNWeights::forward (model.rs:713-735): hidden = silu(x . Wg^T) * (x . Wu^T),
    out = hidden . Wd^T, silu(v) = v / (1 + exp(-v)) (model.rs:1187-1189).  The
    engine's fused_gemm_silu (gemm_engine/vulkan_backend.rs:111-131) has the same
    meaning, silu(gate) * up; here gate and up share one launch that writes `hidden` directly;
  * prepare_qkv (model.rs:1379-1410): q, k, v = linear_gemm(x, W_{q,k,v})
    (model.rs:1392-1394), here one launch for the three.  CachedAttention runs them
    together with the step that lies between them and o_proj (attention.py).

The host-array methods are synchronous and mirror the reference's signatures; from
the weight's gemm_min_rows() rows on (prefill: 64-128 rows by the weight's shape)
they run the fp32-activation GEMMs, below it (and for
Q4_1 / Q5_K weights, whose blocks carry a minimum) the decode GEMVs.  The *_device methods take device buffers and a stream and only enqueue
work.
"""
from __future__ import annotations

import ctypes

import numpy as np

from ._native import check, lib
from .attention import DType, KVCache, PagedAttention, Rope, StepPlan
from .ops import DeviceBuffer, InvalidInput, QuantizedWeight, gemm_f32_workspace

MAX_GROUP = 4  # weights per gemv_multi launch


def gemv_multi(weights, d_x: DeviceBuffer, d_ys, batch: int, stream=None) -> None:
    """d_ys[i][batch, N_i] = x[batch, K] . W_i^T for up to 4 weights of one type and K."""
    n = len(weights)
    if n != len(d_ys):
        raise InvalidInput(f"{n} weights but {len(d_ys)} outputs")
    hs = (ctypes.c_void_p * max(n, 1))(*[w.handle.value for w in weights])
    ys = (ctypes.c_void_p * max(n, 1))(*[y.ptr.value for y in d_ys])
    check(lib().openmini_qmm_gemv_multi(hs, n, d_x.ptr, ys, int(batch), stream))


def ffn_gate_up(gate: QuantizedWeight, up: QuantizedWeight, d_x: DeviceBuffer, d_h: DeviceBuffer,
                batch: int, stream=None) -> None:
    """d_h[batch, N] = silu(x . Wg^T) * (x . Wu^T), fp32 activations (decode)."""
    check(lib().openmini_qmm_ffn_gate_up(gate.handle, up.handle, d_x.ptr, d_h.ptr, int(batch), stream))


def ffn_gate_up_bf16(gate: QuantizedWeight, up: QuantizedWeight, d_x: DeviceBuffer,
                     d_h: DeviceBuffer, m: int, stream=None) -> None:
    """The same with bf16 activations (raw bits) on the prefill GEMM."""
    check(lib().openmini_qmm_ffn_gate_up_bf16(gate.handle, up.handle, d_x.ptr, d_h.ptr, int(m), stream))


def ffn_gate_up_f32(gate: QuantizedWeight, up: QuantizedWeight, d_x: DeviceBuffer, d_h: DeviceBuffer,
                    m: int, d_work: DeviceBuffer, stream=None) -> None:
    """The same with fp32 activations on the prefill GEMM (x split once into d_work,
    gemm_f32_workspace(m, K) bytes)."""
    check(lib().openmini_qmm_ffn_gate_up_f32(gate.handle, up.handle, d_x.ptr, d_h.ptr, int(m), d_work.ptr,
                                             d_work.nbytes, stream))


def _rows(x: np.ndarray, k: int) -> np.ndarray:
    x = np.ascontiguousarray(x, dtype=np.float32)
    if x.ndim != 2 or x.shape[1] != k or x.shape[0] < 1:
        raise InvalidInput(f"x shape {x.shape} does not match K = {k}")
    return x


class FFNWeights:
    """FFNWeights (model.rs:706-711) holding quantized gate / up / down projections:
    gate_proj, up_proj [intermediate, hidden], down_proj [hidden, intermediate]."""

    def __init__(self, gate_proj: QuantizedWeight, up_proj: QuantizedWeight,
                 down_proj: QuantizedWeight):
        if (gate_proj.n_rows, gate_proj.k_cols) != (up_proj.n_rows, up_proj.k_cols):
            raise InvalidInput("gate_proj and up_proj differ in shape")
        if down_proj.k_cols != gate_proj.n_rows:
            raise InvalidInput(f"down_proj K = {down_proj.k_cols} != intermediate {gate_proj.n_rows}")
        self.gate_proj, self.up_proj, self.down_proj = gate_proj, up_proj, down_proj

    @property
    def hidden_size(self) -> int:
        return self.gate_proj.k_cols

    @property
    def intermediate_size(self) -> int:
        return self.gate_proj.n_rows

    def forward_device(self, d_x: DeviceBuffer, d_h: DeviceBuffer, d_out: DeviceBuffer, batch: int,
                       stream=None) -> None:
        """out[batch, hidden] = (silu(x . Wg^T) * (x . Wu^T)) . Wd^T with fp32
        activations: one gate/up launch and one down launch per 4 rows; d_h
        [batch, intermediate] fp32 is the caller's scratch."""
        ffn_gate_up(self.gate_proj, self.up_proj, d_x, d_h, batch, stream)
        self.down_proj.gemv(d_h, d_out, batch, stream)

    def forward(self, x: np.ndarray) -> np.ndarray:
        """model.rs:713-735 on host arrays: x [seq, hidden] -> [seq, hidden]."""
        x = _rows(x, self.hidden_size)
        m = x.shape[0]
        d_x = DeviceBuffer.from_numpy(x)
        d_h = DeviceBuffer(m * self.intermediate_size * 4)
        d_out = DeviceBuffer(m * self.down_proj.n_rows * 4)
        pair_gemm, down_gemm = self.gate_proj.prefill_gemm(m), self.down_proj.prefill_gemm(m)
        if not pair_gemm and not down_gemm:
            self.forward_device(d_x, d_h, d_out, m)
        else:
            work = gemm_f32_workspace(m, max(self.hidden_size, self.intermediate_size))
            if pair_gemm:
                ffn_gate_up_f32(self.gate_proj, self.up_proj, d_x, d_h, m, work)
            else:
                ffn_gate_up(self.gate_proj, self.up_proj, d_x, d_h, m)
            if down_gemm:
                self.down_proj.gemm_f32(d_h, d_out, m, work)
            else:
                self.down_proj.gemv(d_h, d_out, m)
        return d_out.download(np.float32, (m, self.down_proj.n_rows))

    def hidden(self, x: np.ndarray) -> np.ndarray:
        """silu(x . Wg^T) * (x . Wu^T), the input of down_proj (model.rs:728-730)."""
        x = _rows(x, self.hidden_size)
        m = x.shape[0]
        d_x = DeviceBuffer.from_numpy(x)
        d_h = DeviceBuffer(m * self.intermediate_size * 4)
        if self.gate_proj.prefill_gemm(m):
            ffn_gate_up_f32(self.gate_proj, self.up_proj, d_x, d_h, m, gemm_f32_workspace(m, self.hidden_size))
        else:
            ffn_gate_up(self.gate_proj, self.up_proj, d_x, d_h, m)
        return d_h.download(np.float32, (m, self.intermediate_size))


class AttentionWeights:
    """AttentionWeights (model.rs:696-703) holding quantized q / k / v / o projections
    (o_proj may be None when only the input projections are needed)."""

    def __init__(self, q_proj: QuantizedWeight, k_proj: QuantizedWeight, v_proj: QuantizedWeight,
                 o_proj: QuantizedWeight | None = None):
        for w in (k_proj, v_proj):
            if w.k_cols != q_proj.k_cols or w.tensor_type != q_proj.tensor_type:
                raise InvalidInput("q/k/v projections must share K and type")
        self.q_proj, self.k_proj, self.v_proj, self.o_proj = q_proj, k_proj, v_proj, o_proj

    def project_qkv_device(self, d_x: DeviceBuffer, d_q: DeviceBuffer, d_k: DeviceBuffer,
                           d_v: DeviceBuffer, batch: int, stream=None) -> None:
        gemv_multi((self.q_proj, self.k_proj, self.v_proj), d_x, (d_q, d_k, d_v), batch, stream)

    def project_qkv(self, x: np.ndarray):
        """The three linear_gemm calls of prepare_qkv (model.rs:1392-1394) before RoPE:
        x [seq, hidden] -> (q [seq, Nq], k [seq, Nk], v [seq, Nv])."""
        x = _rows(x, self.q_proj.k_cols)
        m = x.shape[0]
        d_x = DeviceBuffer.from_numpy(x)
        ws = (self.q_proj, self.k_proj, self.v_proj)
        outs = [DeviceBuffer(m * w.n_rows * 4) for w in ws]
        if self.q_proj.prefill_gemm(m):
            work = gemm_f32_workspace(m, self.q_proj.k_cols)
            for w, o in zip(ws, outs):
                w.gemm_f32(d_x, o, m, work)
        else:
            self.project_qkv_device(d_x, *outs, m)
        return tuple(o.download(np.float32, (m, w.n_rows)) for o, w in zip(outs, ws))

    def project_o(self, attn: np.ndarray) -> np.ndarray:
        """attn [seq, heads * head_dim] . Wo^T."""
        if self.o_proj is None:
            raise InvalidInput("no o_proj")
        attn = _rows(attn, self.o_proj.k_cols)
        m = attn.shape[0]
        d_a = DeviceBuffer.from_numpy(attn)
        d_o = DeviceBuffer(m * self.o_proj.n_rows * 4)
        if self.o_proj.prefill_gemm(m):
            self.o_proj.gemm_f32(d_a, d_o, m)
        else:
            self.o_proj.gemv(d_a, d_o, m)
        return d_o.download(np.float32, (m, self.o_proj.n_rows))


class CachedAttention:
    """One layer's attention over its paged cache: the q / k / v projections, rotary
    positions and the cache write, attention, and the output projection,
    for any mix of decoding requests and short prompts (a prompt's tokens are rows of their
    own, each seeing the keys up to its position).

    `attention` may be shared by layers that run one after the other; buffers for up to
    max_tokens rows are allocated here."""

    def __init__(self, weights: AttentionWeights, rope: Rope, cache: KVCache, q_heads: int, max_tokens: int,
                 q_dtype: DType = DType.BF16, attention: PagedAttention | None = None):
        head_dim = cache.head_dim
        if weights.o_proj is None:
            raise InvalidInput("no o_proj")
        if (weights.q_proj.n_rows, weights.k_proj.n_rows, weights.v_proj.n_rows, weights.o_proj.k_cols) != \
                (q_heads * head_dim, cache.kv_heads * head_dim, cache.kv_heads * head_dim, q_heads * head_dim):
            raise InvalidInput(f"projections do not have {q_heads} query and {cache.kv_heads} key heads of {head_dim}")
        self.weights, self.rope, self.cache = weights, rope, cache
        self.q_heads, self.max_tokens, self.q_dtype = int(q_heads), int(max_tokens), DType(q_dtype)
        self.attention = attention or PagedAttention(q_heads, cache.kv_heads, head_dim, q_dtype, DType.F32)
        q, kv = q_heads * head_dim, cache.kv_heads * head_dim
        self.d_q, self.d_k, self.d_v = (DeviceBuffer(max_tokens * n * 4) for n in (q, kv, kv))
        self.d_q16, self.d_attn = DeviceBuffer(max_tokens * q * 2), DeviceBuffer(max_tokens * q * 4)

    @property
    def attention(self) -> PagedAttention:
        return self._attention

    @attention.setter
    def attention(self, shared: PagedAttention) -> None:
        if shared.q_dtype != self.q_dtype or shared.out_dtype != DType.F32:
            raise InvalidInput("the shared attention has other types")
        theirs, ours = (shared.q_heads, shared.kv_heads, shared.head_dim), (self.q_heads, self.cache.kv_heads, self.cache.head_dim)
        if theirs != ours:
            raise InvalidInput(f"the shared attention has heads {theirs}, the layer {ours}")
        self._attention = shared

    def forward_device(self, d_x: DeviceBuffer, plan: StepPlan, d_tables, requests: int, tokens: int, d_out: DeviceBuffer,
                       d_positions=None, stream=None, max_pages: int | None = None) -> None:
        """d_out [tokens, hidden] for the step that `plan` laid out (plan.run on the same
        stream before the first layer): d_x [tokens, hidden] fp32, d_tables the tables that
        the plan filled.  d_positions [axes][tokens]: None takes the plan's, for a rope of one
        axis (of several, text too has its position on each).
        max_pages: columns that the step's longest request needs, where that is known (None:
        the tables' width); attention of short rows is faster for it."""
        most = plan.max_pages if max_pages is None else int(max_pages)
        if not 0 < most <= plan.max_pages:
            raise InvalidInput(f"max_pages {most}, tables of {plan.max_pages}")
        if tokens > min(self.max_tokens, plan.max_tokens):
            raise InvalidInput(f"{tokens} tokens, planned for {min(self.max_tokens, plan.max_tokens)}")
        if plan.page_size != self.cache.page_size:
            raise InvalidInput(f"plan for pages of {plan.page_size} tokens, the cache's have {self.cache.page_size}")
        for name, buf, columns in (("d_x", d_x, self.weights.q_proj.k_cols), ("d_out", d_out, self.weights.o_proj.n_rows)):
            if buf.nbytes < 4 * tokens * columns:
                raise InvalidInput(f"{name} holds {buf.nbytes} bytes, {4 * tokens * columns} are needed")
        if d_positions is None and self.rope.n_axes > 1:
            raise InvalidInput(f"the plan's positions are for one axis, the rope has {self.rope.n_axes}")
        w = self.weights
        w.project_qkv_device(d_x, self.d_q, self.d_k, self.d_v, tokens, stream)
        self.rope.append(self.cache, self.d_q, self.d_k, self.d_v, DType.F32, self.d_q16, self.q_dtype,
                         plan.positions if d_positions is None else d_positions, plan.slots, tokens, self.q_heads, stream)
        self.attention.run(self.cache, self.d_q16, self.d_attn, d_tables, most, plan.row_lens, tokens,
                           d_rows=plan.rows, requests=requests, table_stride=plan.max_pages, stream=stream)
        w.o_proj.gemv(self.d_attn, d_out, tokens, stream)


__all__ = ["AttentionWeights", "CachedAttention", "FFNWeights", "MAX_GROUP", "ffn_gate_up", "ffn_gate_up_bf16",
           "ffn_gate_up_f32", "gemv_multi"]
