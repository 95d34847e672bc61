"""`FusedKernels` (FusedKernels.swift:7-286) on the HIP library.

Same method names and argument meaning as the Swift class; tensors are torch
GPU tensors, outputs are allocated by the callee (as MLX's
`outputShapes`/`outputDTypes`), and shape misuse raises GlinerDecideError
instead of trapping.  The default-graph kernels the encoder runs (fused
relative bias + masked softmax + P.V, embedding LayerNorm, linear epilogues)
are exposed beside them.
"""

from __future__ import annotations

import math

import torch

from . import _native as N
from .device import as_f16, as_i32, call_on, dtype16, ptr, same_kind, stream_handle


def _dims(t: torch.Tensor, n: int, name: str):
    if t.dim() != n:
        raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"{name} must have {n} dimensions (got {tuple(t.shape)})")
    return tuple(t.shape)


def _indices(c2p_indices, p2c_indices, H: int, L: int):
    """General index tensors broadcast to [H, L, L], or (None, None) for the
    closed form."""
    if c2p_indices is None and p2c_indices is None:
        return None, None
    if c2p_indices is None or p2c_indices is None:
        raise N.GlinerDecideError(N.GD_ERR_INVALID_ARGUMENT, "give both index tensors, or neither")
    return _index_tensor(c2p_indices, "c2p_indices", H, L), _index_tensor(p2c_indices, "p2c_indices", H, L)


def _index_tensor(t: torch.Tensor, name: str, H: int, L: int) -> torch.Tensor:
    t = as_i32(t, name)
    return t if t.shape == (H, L, L) else t.expand(1, H, L, L).reshape(H, L, L).contiguous()


def _shaped(t: torch.Tensor, name: str, *shape: int) -> torch.Tensor:
    t = as_f16(t, name)
    return t if t.shape == shape else t.reshape(shape).contiguous()


_OUTPUTS = {"probs": N.GD_ATTN_OUT_PROBS, "context": N.GD_ATTN_OUT_CONTEXT, "bias": N.GD_ATTN_OUT_BIAS}
_SCORES = {"default": N.GD_ATTN_SCORE_DEFAULT, "explicit": N.GD_ATTN_SCORE_EXPLICIT,
           "kernel_bias": N.GD_ATTN_SCORE_KERNEL_BIAS, "kernel_bias_explicit": N.GD_ATTN_SCORE_KERNEL_BIAS_EXPLICIT,
           "fused": N.GD_ATTN_SCORE_FUSED}
_MASKS = {"attention": N.GD_MASK_ATTENTION, "additive": N.GD_MASK_ADDITIVE}
_EPILOGUES = {"none": N.GD_EPI_NONE, "bias": N.GD_EPI_BIAS, "gelu": N.GD_EPI_BIAS_GELU, "relu": N.GD_EPI_BIAS_RELU}
_ACTIVATIONS = {"none": N.GD_ACT_NONE, "relu": N.GD_ACT_RELU, "gelu": N.GD_ACT_GELU,
                "gelu_tanh": N.GD_ACT_GELU_TANH, "silu": N.GD_ACT_SILU}
_NORMS = {"layer": N.GD_NORM_LAYER, "rms": N.GD_NORM_RMS}


_NO_ROWS = N.GdRows(None, 0)


def _choice(table: dict, key, name: str) -> int:
    code = table.get(key)
    if code is None:
        raise N.GlinerDecideError(N.GD_ERR_INVALID_ARGUMENT, f"{name} must be one of {', '.join(table)} (got {key!r})")
    return code


def _tokens(t: torch.Tensor, name: str) -> N.GdTokens:
    """[T, H, D] with contiguous D; a stride that no element uses is 0."""
    if t.dim() == 3:
        T, H, D = t.shape
        st, sh, sd = t.stride()
        if sd == 1 or D <= 1:
            return N.GdTokens(t.data_ptr(), st if T > 1 else 0, sh if H > 1 else 0)
    raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"{name} must be a [tokens, heads, head_dim] view with contiguous "
                                              f"head_dim (got {tuple(t.shape)}, strides {t.stride()})")


def _rows(t: torch.Tensor, cols: int):
    """(tensor, GdRows) of t [..., cols] as rows with contiguous, non-overlapping columns (copied where t has none)."""
    if not t.is_contiguous():
        if t.dim() != 2:
            t = t.reshape(-1, cols) if cols else t.reshape(math.prod(t.shape[:-1]), 0)
        many = t.shape[0] > 1
        if (cols <= 1 or t.stride(1) == 1) and (not many or t.stride(0) >= cols):
            return t, N.GdRows(t.data_ptr(), t.stride(0) if many else cols)
        t = t.contiguous()
    return t, N.GdRows(t.data_ptr(), cols)


def _vector(t: torch.Tensor | None, like: torch.Tensor, shape: tuple, name: str) -> torch.Tensor | None:
    if t is None:
        return None
    if t.dtype is like.dtype and t.get_device() == like.get_device() and t.shape == shape and t.is_contiguous():
        return t
    same_kind(t, like, name)
    if t.shape != shape:
        raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"{name} must be {list(shape)} (got {tuple(t.shape)})")
    return t.contiguous()


def _data(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _output(out: torch.Tensor, like: torch.Tensor, shape, name: str) -> int:
    """Row stride of a given output; refuses one whose rows (last axis) are not contiguous at one stride."""
    same_kind(out, like, name)
    if out.shape != shape:
        raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"{name} must be {tuple(shape)} (got {tuple(out.shape)})")
    if out.is_contiguous():
        return shape[-1]
    if out.dim() != 2 or (out.shape[1] > 1 and out.stride(1) != 1):
        raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"{name} must be contiguous, or rows with contiguous columns")
    return out.stride(0) if out.shape[0] > 1 else shape[-1]


class FusedKernels:
    """Mirror of `FusedKernels` (FusedKernels.swift:7)."""

    def __init__(self):
        self._lib = N.lib()

    # -- FusedKernels.residualLayerNorm (FusedKernels.swift:261-286) --------
    def residual_layer_norm(self, x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                            bias: torch.Tensor, eps: float, round_sum_f16: bool = False) -> torch.Tensor:
        """LayerNorm(x + residual) * weight + bias over the last axis.

        round_sum_f16=False keeps x + residual in fp32 (the Metal kernel);
        True rounds it to fp16 first (the default graph `norm(x + residual)`,
        DeBERTa.swift:463).  residual=None gives a plain LayerNorm."""
        x = as_f16(x, "x")
        if residual is not None:
            residual = as_f16(residual, "residual")
            if residual.shape != x.shape:
                raise N.GlinerDecideError(N.GD_ERR_SHAPE, "residual shape mismatch")
        if x.dim() < 1:
            raise N.GlinerDecideError(N.GD_ERR_SHAPE, "x must have at least one dimension")
        cols = x.shape[-1]
        rows = x.numel() // cols if cols else 0
        weight = as_f16(weight, "weight")
        bias = as_f16(bias, "bias")
        out = torch.empty_like(x)
        N.check(self._lib.gd_residual_layer_norm(ptr(x), ptr(residual), ptr(weight), ptr(bias), ptr(out), rows, cols,
                                                 float(eps), N.GD_LN_SUM_F16 if round_sum_f16 else 0,
                                                 stream_handle()))
        return out

    # -- FusedKernels.relativeBias (FusedKernels.swift:214-258) -------------
    def relative_bias(self, q, k, position_key, position_query, c2p_indices, p2c_indices, key_mask, scale: float,
                      batch: int, heads: int, sequence_length: int, head_dimension: int,
                      position_count: int) -> torch.Tensor:
        """(q.posK[c2p] + k.posQ[p2c]) * scale with masked keys := -65504,
        general index tensors [1 or H, L, L]; returns [B, H, L, L] fp16.
        c2p_indices = p2c_indices = None selects the closed-form indices
        (the ones the classifier builds) on the MFMA attention kernel."""
        q = as_f16(q, "q")
        k = as_f16(k, "k")
        if q.shape != k.shape or q.dim() != 4 or q.shape[2] != sequence_length or q.shape[3] != head_dimension:
            raise N.GlinerDecideError(N.GD_ERR_SHAPE, "q/k must both be [B, H, L, D]")
        H, L = heads, sequence_length
        c2p, p2c = _indices(c2p_indices, p2c_indices, H, L)
        pk = _shaped(position_key, "position_key", H, position_count, head_dimension)
        pq = _shaped(position_query, "position_query", H, position_count, head_dimension)
        km = _shaped(key_mask, "key_mask", batch, L)
        out = torch.empty((batch, H, L, L), dtype=torch.float16, device=q.device)
        N.check(self._lib.gd_relative_bias(ptr(q), ptr(k), ptr(pk), ptr(pq), ptr(c2p), ptr(p2c), ptr(km),
                                           float(scale), batch, H, L, head_dimension, position_count, ptr(out),
                                           stream_handle()))
        return out

    # -- FusedKernels.fusedAttention (FusedKernels.swift:160-210) -----------
    def fused_attention(self, queries, keys, values, position_key, position_query, c2p_indices, p2c_indices,
                        key_mask, scale: float, batch: int, heads: int, sequence_length: int, head_dimension: int,
                        position_count: int) -> torch.Tensor:
        """Whole attention with general indices (None for the closed form, on
        the MFMA attention kernel); returns [B, L, H, D] fp16."""
        q = as_f16(queries, "queries")
        k = as_f16(keys, "keys")
        v = as_f16(values, "values")
        if not (q.shape == k.shape == v.shape) or q.dim() != 4:
            raise N.GlinerDecideError(N.GD_ERR_SHAPE, "queries/keys/values must all be [B, H, L, D]")
        if tuple(q.shape) != (batch, heads, sequence_length, head_dimension):
            raise N.GlinerDecideError(N.GD_ERR_SHAPE, "queries shape does not match the given dimensions")
        H, L = heads, sequence_length
        c2p, p2c = _indices(c2p_indices, p2c_indices, H, L)
        pk = _shaped(position_key, "position_key", H, position_count, head_dimension)
        pq = _shaped(position_query, "position_query", H, position_count, head_dimension)
        km = _shaped(key_mask, "key_mask", batch, L)
        out = torch.empty((batch, L, H, head_dimension), dtype=torch.float16, device=q.device)
        N.check(self._lib.gd_fused_attention(ptr(q), ptr(k), ptr(v), ptr(pk), ptr(pq), ptr(c2p), ptr(p2c), ptr(km),
                                             float(scale), batch, H, L, head_dimension, position_count, ptr(out),
                                             stream_handle()))
        return out

    # -- default graph: relative bias + masked softmax (+ P.V) --------------
    def deberta_attention(self, q, k, v, position_key, position_query, mask, *, output: str = "context",
                          mask_kind: str = "attention", out: torch.Tensor | None = None,
                          score: str = "default") -> torch.Tensor:
        """Closed-form-index DeBERTa attention (DeBERTa.swift:322-410).

        q, k, v: [B, H, L, D] views with contiguous D (any strides, e.g. the
        split of a fused [B, L, 3, H, D] projection); position_key /
        position_query: [H, P, D] views with contiguous D; mask: [B, L] fp16.
        output: "probs" -> [B, H, L, L]; "context" -> [B, L, H*D];
        "bias" -> the SDPA additive mask [B, H, L, L] (or the kernel bias).
        score: the graph reproduced -- "default" (:374-394), "explicit"
        (useFastAttention = false, :397-409), "kernel_bias"
        (useCustomRelativeKernel, :357-372 + SDPA), "kernel_bias_explicit"
        (both), "fused" (useFusedAttentionKernel, :337-354)."""
        for name, t in (("q", q), ("k", k)) + ((("v", v),) if v is not None else ()):
            if not t.is_cuda or t.dtype != torch.float16 or t.dim() != 4 or t.stride(3) != 1:
                raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"{name} must be a [B, H, L, D] fp16 GPU view with "
                                                          "contiguous D")
        B, H, L, D = q.shape
        for name, t in (("position_key", position_key), ("position_query", position_query)):
            if t.dim() != 3 or t.shape[0] != H or t.shape[2] != D or t.stride(2) != 1 or t.dtype != torch.float16:
                raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"{name} must be a [H, P, D] fp16 view with contiguous D")
        P = position_key.shape[1]
        mask = _shaped(mask, "mask", B, L)
        kind, sc, mk = _OUTPUTS[output], _SCORES[score], _MASKS[mask_kind]
        if out is None:
            shape = (B, L, H * D) if kind == N.GD_ATTN_OUT_CONTEXT else (B, H, L, L)
            out = torch.empty(shape, dtype=torch.float16, device=q.device)
        ldo = H * D if kind == N.GD_ATTN_OUT_CONTEXT else L
        vv = v if v is not None else q
        N.check(self._lib.gd_deberta_attention(
            N.GdBhld(ptr(q), *q.stride()[:3]), N.GdBhld(ptr(k), *k.stride()[:3]),
            N.GdBhld(ptr(vv), *vv.stride()[:3]),
            N.GdTable(ptr(position_key), position_key.stride(0), position_key.stride(1)),
            N.GdTable(ptr(position_query), position_query.stride(0), position_query.stride(1)),
            ptr(mask), mk, B, H, L, D, P, 256, kind | sc, ptr(out), ldo, stream_handle()))
        return out

    # -- default graph: embedding stage (DeBERTa.swift:285-292) -------------
    def embedding_layer_norm(self, ids, attention_mask, table, gamma, beta, eps: float,
                             error_flag: torch.Tensor | None = None) -> torch.Tensor:
        ids = as_i32(ids, "ids")
        B, L = _dims(ids, 2, "ids")
        mask = as_f16(attention_mask, "attention_mask").reshape(B, L).contiguous()
        table = as_f16(table, "table")
        V, Cdim = _dims(table, 2, "table")
        out = torch.empty((B, L, Cdim), dtype=torch.float16, device=ids.device)
        N.check(self._lib.gd_embedding_layer_norm(ptr(ids), ptr(mask), ptr(table), ptr(as_f16(gamma, "gamma")),
                                                  ptr(as_f16(beta, "beta")), ptr(out), B, L, Cdim, V, float(eps),
                                                  ptr(error_flag), stream_handle()))
        return out

    # -- LinearWeight / FusedProjectionWeight (DeBERTa.swift:60-92) ---------
    def linear(self, x, weight, bias=None, epilogue: str = "bias", rows: torch.Tensor | None = None) -> torch.Tensor:
        """epilogue(x W^T + b); epilogue in {"none", "bias", "gelu", "relu"}.
        rows (int32) gathers rows of x first (marker gather)."""
        x = as_f16(x, "x")
        w = as_f16(weight, "weight")
        N_, K = _dims(w, 2, "weight")
        if x.shape[-1] != K:
            raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"x last dim {x.shape[-1]} != weight in-features {K}")
        x2 = x if x.dim() == 2 else x.reshape(-1, K)
        if rows is not None:
            rows = as_i32(rows, "rows")
            M = rows.numel()
            lead = (M,)
        else:
            M = x2.shape[0]
            lead = tuple(x.shape[:-1])
        epi = _EPILOGUES[epilogue]
        b = as_f16(bias, "bias") if bias is not None else None
        out = torch.empty(lead + (N_,), dtype=torch.float16, device=x.device)
        N.check(self._lib.gd_linear(ptr(x2), ptr(w), ptr(b), ptr(out), M, N_, K, K, N_, ptr(rows), x2.shape[0], epi,
                                    stream_handle()))
        return out

    # -- a block over packed rows (no counterpart in the reference) ---------
    def packed_attention(self, q, k, v, q_offsets, k_offsets=None, *, scale: float | None = None, causal: bool = True,
                         out: torch.Tensor | None = None) -> torch.Tensor:
        """Softmax attention over packed sequences with grouped heads, fp16 or bf16.

        q: [Tq, H, D], k and v: [Tk, Hk, D] views with contiguous D (the parts
        of one projection's output, say), H a multiple of Hk, D one of 32, 64,
        96, 128, 192, 256; head h reads key head h // (H // Hk).  Sequence b
        holds queries q_offsets[b]:q_offsets[b+1] and keys
        k_offsets[b]:k_offsets[b+1] (integer GPU tensors [B + 1] that do not
        decrease; None: the keys are the queries' own tokens).  causal: query i
        of nq sees the keys j <= nk - nq + i, the last one all of them; a
        query that sees none gets 0.  scale: of q . k, 1 / sqrt(D) by default.

        Returns [Tq, H, D]; rows of no sequence are 0, in a given `out` (heads
        contiguous, overlapping no input) they are left as they were.  Forward
        only: the result carries no gradient."""
        dtype = dtype16(q, "q")
        qt, kt, vt = _tokens(q, "q"), _tokens(k, "k"), _tokens(v, "v")
        qd, dev = q.dtype, q.get_device()
        if k.dtype is not qd or v.dtype is not qd or k.get_device() != dev or v.get_device() != dev:
            same_kind(k, q, "k")
            same_kind(v, q, "v")
        Tq, H, D = q.shape
        Tk, Hk, Dk = k.shape
        if k.shape != v.shape or Dk != D or D == 0:
            raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"k and v must both be [tokens, kv_heads, {D}]")
        q_offsets, batch = self._offsets(q_offsets, q, "q_offsets")
        if k_offsets is not None:
            k_offsets, kb = self._offsets(k_offsets, q, "k_offsets")
            if kb != batch:
                raise N.GlinerDecideError(N.GD_ERR_SHAPE, "q_offsets and k_offsets must have one length")
        flags = N.GD_PACKED_CAUSAL if causal else 0
        if out is None:
            out = torch.empty_like(q) if q.is_contiguous() else torch.empty((Tq, H, D), dtype=qd, device=q.device)
            ldo = H * D
            flags |= N.GD_PACKED_ZERO_REST
        else:
            same_kind(out, q, "out")
            if out.shape != q.shape or (out.numel() and (out.stride(2) != 1 or (H > 1 and out.stride(1) != D))):
                raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"out must be {tuple(q.shape)} with contiguous heads")
            ldo = out.stride(0) if Tq > 1 else H * D
        need = self._lib.gd_packed_attention_workspace(batch, Tq, Tk, H, Hk, D)
        work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        call_on(q, self._lib.gd_packed_attention, qt, kt, vt, q_offsets.data_ptr(), _data(k_offsets), batch, Tq, Tk, H,
                Hk, D, dtype, D ** -0.5 if scale is None else scale, flags, out.data_ptr(), ldo, _data(work), need)
        return out

    @staticmethod
    def _offsets(t: torch.Tensor, like: torch.Tensor, name: str):
        if t.get_device() != like.get_device():
            raise ValueError(f"{name} must be on {like.device} (got {t.device})")
        if t.dtype is not torch.int32 or not t.is_contiguous():
            t = as_i32(t, name)
        if t.dim() != 1 or t.numel() < 1:
            raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"{name} must be [batch + 1] (got {tuple(t.shape)})")
        return t, t.numel() - 1

    def projection(self, x, weight, bias=None, residual=None, *, activation: str = "none", scale: float = 1.0,
                   out: torch.Tensor | None = None) -> torch.Tensor:
        """residual + scale * act(x W^T + bias), fp16 or bf16, rounded once.

        x: [..., K], weight: [N, K] (rows at any stride), bias: [N], residual:
        [..., N]; activation in {"none", "relu", "gelu", "gelu_tanh", "silu"}.
        Any sizes; rows of 16-byte alignment run faster.  `out` may be the
        residual itself and overlaps nothing else.  Forward only."""
        dtype = dtype16(x, "x")
        same_kind(weight, x, "weight")
        n, K = _dims(weight, 2, "weight")
        xs = x.shape
        if not xs or xs[-1] != K:
            raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"x {tuple(xs)} does not end in the weight's {K} columns")
        act = _choice(_ACTIVATIONS, activation, "activation")
        shape = (xs[0], n) if len(xs) == 2 else (*xs[:-1], n)
        x2, xr = _rows(x, K)
        w2, wr = _rows(weight, K)
        bias = _vector(bias, x, (n,), "bias")
        res = _NO_ROWS
        if residual is not None:
            same_kind(residual, x, "residual")
            if residual.shape != shape:
                raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"residual must be {shape} (got {tuple(residual.shape)})")
            residual, res = _rows(residual, n)
        if out is None:
            out, ldo = torch.empty(shape, dtype=x.dtype, device=x.device), n
        else:
            ldo = _output(out, x, shape, "out")
        call_on(x, self._lib.gd_projection, xr, wr, _data(bias), res, out.data_ptr(), ldo,
                x.numel() // K if K else 0, n, K, act, float(scale), dtype)
        return out

    def block_norm(self, y, residual, *, pre_weight, pre_bias=None, post_weight=None, post_bias=None, gate=None,
                   scale: float = 1.0, eps: float = 1e-6, kind: str = "rms", out=None):
        """(h, n) with h = residual + scale * gate * post(y) and n = pre(h): the
        norm after a block, its gate and residual scale and the norm before the
        next block in one pass.

        y: [..., C] fp16 or bf16; residual: its shape, its type or fp32 (h has
        the residual's type, n has y's); kind "rms" or "layer" for both norms;
        post_weight=None leaves the first norm out; gate: any shape that
        broadcasts to y's and keeps C ([C], [B, 1, C] for [B, L, C], y's own).
        out = (h, n) may be the residual and y themselves.  Forward only."""
        dtype = dtype16(y, "y")
        f32 = residual.dtype is torch.float32
        same_kind(residual, y, "residual", torch.float32 if f32 else None)
        shape = y.shape
        if y.dim() < 1 or residual.shape != shape:
            raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"y {tuple(shape)} and residual {tuple(residual.shape)} differ")
        C = shape[-1]
        rows = y.numel() // C if C else 0
        code = _choice(_NORMS, kind, "kind")
        if pre_weight is None:
            raise N.GlinerDecideError(N.GD_ERR_INVALID_ARGUMENT, "pre_weight is needed")
        vec = (C,)
        pre_w = _vector(pre_weight, y, vec, "pre_weight")
        pre_b = None if pre_bias is None else _vector(pre_bias, y, vec, "pre_bias")
        post_w = None if post_weight is None else _vector(post_weight, y, vec, "post_weight")
        post_b = None if post_bias is None else _vector(post_bias, y, vec, "post_bias")
        y2, yr = _rows(y, C)
        r2, rr = _rows(residual, C)
        g, per_gate = _NO_ROWS, 1
        if gate is not None:
            same_kind(gate, y, "gate")
            gate, per_gate = self._gate_rows(gate, shape, rows)
            gate, g = _rows(gate, C)
        if out is None:
            # (r2 and y2 are rows: contiguous ones need no format named)
            h = torch.empty_like(r2) if r2 is residual and r2.is_contiguous() else torch.empty(
                shape, dtype=residual.dtype, device=y.device)
            n = torch.empty_like(y2) if y2 is y and y2.is_contiguous() else torch.empty(
                shape, dtype=y.dtype, device=y.device)
            ldh = ldn = C
        else:
            h, n = out
            ldh, ldn = _output(h, r2, shape, "out[0]"), _output(n, y2, shape, "out[1]")
        call_on(y, self._lib.gd_block_norm, yr, rr, g, per_gate, _data(post_w), _data(post_b), _data(pre_w), _data(pre_b),
                h.data_ptr(), ldh, n.data_ptr(), ldn, rows, C, float(eps), float(scale), code, dtype,
                N.GD_F32 if f32 else dtype)
        return h, n

    @staticmethod
    def _gate_rows(gate: torch.Tensor, shape, rows: int):
        """A gate that broadcasts to `shape`, as G rows of its last axis with row r's gate at r // (rows // G), and
        rows // G."""
        if gate.shape == shape:
            return gate, 1
        C = shape[-1]
        if gate.dim() < 1 or gate.dim() > len(shape) or gate.shape[-1] != C:
            raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"gate {tuple(gate.shape)} does not broadcast to {tuple(shape)}")
        if gate.dim() == 1:
            return gate, max(rows, 1)
        lead = (1,) * (len(shape) - gate.dim()) + tuple(gate.shape[:-1])
        if any(a not in (1, b) for a, b in zip(lead, shape[:-1])):
            raise N.GlinerDecideError(N.GD_ERR_SHAPE, f"gate {tuple(gate.shape)} does not broadcast to {tuple(shape)}")
        # its own leading axes first and broadcast ones behind: each gate row serves a run of rows
        own = 0
        while own < len(lead) and lead[own] == shape[own]:
            own += 1
        if any(d != 1 for d in lead[own:]):
            return gate.expand(shape), 1
        return gate.reshape(-1, C), max(rows // max(math.prod(lead), 1), 1)

    def relative_index_table(self, n: int, device=None) -> torch.Tensor:
        """Device-computed idx(r) for r in [-(n-1), n-1] (DeBERTa.swift:521-551)."""
        out = torch.empty(2 * n - 1, dtype=torch.int32, device=device or torch.device("cuda"))
        N.check(self._lib.gd_relative_index_table(ptr(out), n, 256, 512, stream_handle()))
        return out


def scale_f32(head_size: int) -> float:
    """1 / Float(headSize * 3).squareRoot() (DeBERTa.swift:347)."""
    import numpy as np
    return float(np.float32(1.0) / np.float32(math.sqrt(head_size * 3)))
