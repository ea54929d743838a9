"""
Stage 0a: the ColBERT query encoder on the sm_100a kernels of csrc/enc.cu.

Mirrors the reference's fast encoder (src/fast_encoder.py): the same network as a flat
function over fp16 weights -- embeddings + LayerNorm, 12 x [self-attention, LayerNorm, GELU
MLP, LayerNorm], ColBERT's linear 768 -> 128, L2 normalisation -- on fixed [B, 32] token
shapes, captured in one CUDA graph per batch shape.  Every operation runs in
libragrt_b200.so: the seven matrix products per layer on the tensor cores with bias, GELU
and residual fused into their epilogues, the final projection with the fp16 rounding and L2
normalisation fused, LayerNorm and the 32-token attention as their own kernels.

  flat_weights(bert, linear)     the reference's weight dict (fast_encoder.py:31-54)
  flat_forward(W, ids, mask)     [B, L] int64 token ids and attention mask -> [B, L, 128] fp16
  FastQueryEncoder(checkpoint)   encode(text) / encode_batch(texts), as the reference's class
                                 (fast_encoder.py:80-125); `checkpoint` needs .query_tokenizer,
                                 .linear and a BERT model (.bert, .model.bert or .model.LM)

Layer operators for encoders with packed rows, rotary positions, grouped heads and gated
feed-forward blocks (fp16 or bf16, no counterpart in the reference):

  packed_attention(q, k, v, cu_seqlens, causal)      attention over packed sequences
  qk_norm_rope(q, k, cos, sin, positions, ...)       per-head RMS norm + rotary positions
  gated_ffn(x, w_gate, w_up, act)                    act(x w_gate^T) * (x w_up^T)
  gated_ffn_backward(dh, x, w_gate, w_up, ...)       its gradients

The token ids, [Q] marker and [MASK] padding come from the checkpoint's own tokenizer, as in
the reference; `encode_ids` takes already-tokenized input.
"""
import ctypes
import warnings

import torch

from . import _lib
from .weft import _need_cuda, _ptr, _stream

EPI_BIAS, EPI_BIAS_GELU, EPI_BIAS_GELU_TANH, EPI_BIAS_RESIDUAL, EPI_NORM = 0, 1, 2, 3, 4


def bert_and_linear(checkpoint):
    """(BERT model, ColBERT linear) of a ColBERT checkpoint object (fast_encoder.py:22-28)."""
    bert = getattr(checkpoint, "bert", None)
    if bert is None:
        m = checkpoint.model
        bert = getattr(m, "bert", None) or getattr(m, "LM")
    return bert, checkpoint.linear


def flat_weights(bert, linear, dtype=torch.float16, device="cuda"):
    """fp16 weights of a HuggingFace BertModel state dict + ColBERT's linear, with each layer's
    Q, K and V projections stacked into one [3 D, D] matrix (the reference's layout)."""
    sd = {k: v.detach().to(device=device, dtype=dtype).contiguous() for k, v in bert.state_dict().items()}
    cfg = bert.config
    act = getattr(cfg, "hidden_act", "gelu")
    if act not in ("gelu", "gelu_new", "gelu_python", "gelu_pytorch_tanh"):
        raise RuntimeError(f"unsupported activation {act}")
    W = {"emb_word": sd["embeddings.word_embeddings.weight"],
         "emb_pos": sd["embeddings.position_embeddings.weight"],
         "emb_type": sd["embeddings.token_type_embeddings.weight"][0].contiguous(),
         "emb_ln": (sd["embeddings.LayerNorm.weight"], sd["embeddings.LayerNorm.bias"]),
         "heads": cfg.num_attention_heads, "eps": cfg.layer_norm_eps, "act": act,
         "linear": linear.weight.detach().to(device=device, dtype=dtype).contiguous(), "layers": []}
    for i in range(cfg.num_hidden_layers):
        p = f"encoder.layer.{i}."
        g = lambda n: sd[p + n]
        W["layers"].append({
            "qkv_w": torch.cat([g("attention.self.query.weight"), g("attention.self.key.weight"),
                                g("attention.self.value.weight")], 0).contiguous(),
            "qkv_b": torch.cat([g("attention.self.query.bias"), g("attention.self.key.bias"),
                                g("attention.self.value.bias")], 0).contiguous(),
            "o_w": g("attention.output.dense.weight"), "o_b": g("attention.output.dense.bias"),
            "ln1": (g("attention.output.LayerNorm.weight"), g("attention.output.LayerNorm.bias")),
            "i_w": g("intermediate.dense.weight"), "i_b": g("intermediate.dense.bias"),
            "f_w": g("output.dense.weight"), "f_b": g("output.dense.bias"),
            "ln2": (g("output.LayerNorm.weight"), g("output.LayerNorm.bias")),
        })
    return W


def _gemm(a, w, bias, out, epi, residual=None, ws=None):
    M, K = a.shape
    N = w.shape[0]
    nbytes = ws.numel() * ws.element_size() if ws is not None else 0
    _lib.check(_lib.lib().ragrt_enc_gemm(_ptr(a), _ptr(w), _ptr(bias), _ptr(residual), _ptr(out), M, N, K, epi,
                                         _ptr(ws), nbytes, _stream()))
    return out


def _split_workspace(device):
    """Scratch for the K-split products of small batches.  A product is split only while its
    128 x 128 tiles number at most half the SMs, into at most SMs / tiles slices, so the fp32
    partials never exceed SMs x 128 x 128 values (9.7 MB on 148 SMs)."""
    sms = torch.cuda.get_device_properties(device).multi_processor_count
    return torch.empty(sms * 128 * 128, dtype=torch.float32, device=device)


def _gemm_residual_ln(a, w, bias, residual, ln, eps, tmp, out, ws=None):
    M, K = a.shape
    N = w.shape[0]
    nbytes = ws.numel() * ws.element_size() if ws is not None else 0
    _lib.check(_lib.lib().ragrt_enc_gemm_residual_ln(_ptr(a), _ptr(w), _ptr(bias), _ptr(residual), _ptr(ln[0]),
                                                     _ptr(ln[1]), float(eps), _ptr(tmp), _ptr(out), M, N, K,
                                                     _ptr(ws), nbytes, _stream()))
    return out


def _layernorm(x, ln, eps, out):
    _lib.check(_lib.lib().ragrt_enc_layernorm(_ptr(x), _ptr(ln[0]), _ptr(ln[1]), float(eps), _ptr(out), x.shape[0],
                                              x.shape[1], _stream()))
    return out


def flat_forward(W, ids, mask):
    """ids, mask [B, L] (int64, on the weights' device) -> unit ColBERT query vectors
    [B, L, dim] fp16.  Needs L = 32, hidden size 768 and head size 64 (BERT-base)."""
    _need_cuda(ids, mask, W["emb_word"])
    ids = ids.to(torch.int64).contiguous()
    mask = mask.to(torch.int64).contiguous()
    B, L = ids.shape
    if mask.shape != ids.shape or L > W["emb_pos"].shape[0]:
        raise RuntimeError(f"ids / mask must be [B, L] with L <= {W['emb_pos'].shape[0]} positions")
    M = B * L
    D = W["emb_word"].shape[1]
    H = W["heads"]
    eps = W["eps"]
    dev = ids.device
    x = torch.empty(M, D, dtype=torch.float16, device=dev)
    y = torch.empty(M, D, dtype=torch.float16, device=dev)
    ctx = torch.empty(M, D, dtype=torch.float16, device=dev)
    qkv = torch.empty(M, 3 * D, dtype=torch.float16, device=dev)
    h = torch.empty(M, W["layers"][0]["i_w"].shape[0], dtype=torch.float16, device=dev)
    ws = _split_workspace(dev)
    _lib.check(_lib.lib().ragrt_enc_embed(_ptr(ids), _ptr(W["emb_word"]), _ptr(W["emb_pos"]), _ptr(W["emb_type"]),
                                          _ptr(W["emb_ln"][0]), _ptr(W["emb_ln"][1]), float(eps),
                                          W["emb_word"].shape[0], B, L, D, _ptr(x), _stream()))
    gelu = EPI_BIAS_GELU_TANH if W["act"] in ("gelu_new", "gelu_pytorch_tanh") else EPI_BIAS_GELU
    for lw in W["layers"]:
        _gemm(x, lw["qkv_w"], lw["qkv_b"], qkv, EPI_BIAS, ws=ws)
        _lib.check(_lib.lib().ragrt_enc_attention(_ptr(qkv), _ptr(mask), _ptr(ctx), B, L, H, D, _stream()))
        _gemm_residual_ln(ctx, lw["o_w"], lw["o_b"], x, lw["ln1"], eps, y, x, ws=ws)
        _gemm(x, lw["i_w"], lw["i_b"], h, gelu, ws=ws)
        _gemm_residual_ln(h, lw["f_w"], lw["f_b"], x, lw["ln2"], eps, y, x, ws=ws)
    out = torch.empty(M, W["linear"].shape[0], dtype=torch.float16, device=dev)
    _gemm(x, W["linear"], None, out, EPI_NORM, ws=ws)
    return out.view(B, L, -1)


_DTYPES = {torch.float16: 0, torch.bfloat16: 1}
_ACTS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


_bound = None


class _NoBinding:
    """In the place of the host binding where that is not built: answers None to every call, which the Python
    below then serves."""
    packed_attention = qk_norm_rope = gated_ffn = gated_ffn_backward = staticmethod(lambda *args: None)


def _bind():
    """The host binding (csrc/enc_bind.cpp), given the entry points of the loaded library.  It serves the
    calls whose operands can be used as they lie and answers None to the others, which the Python below
    then copies or refuses."""
    global _bound
    if _bound is None:
        L = _lib.lib()
        try:
            from . import _enc_bind
        except ImportError as e:
            warnings.warn(f"the layer operators run without their host binding, at about 10 us more a call: {e} "
                          f"(build it: python -m ragrt_b200.build)", RuntimeWarning, stacklevel=3)
            _bound = _NoBinding
            return _bound
        _enc_bind.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
            L.ragrt_enc_packed_attention, L.ragrt_enc_qk_norm_rope, L.ragrt_enc_gated_ffn,
            L.ragrt_enc_gated_ffn_backward, L.ragrt_enc_gated_ffn_workspace)))
        _bound = _enc_bind
    return _bound


def _dtype16(*ts):
    """Type code of a call's 16-bit tensors (None for an absent one), which must agree."""
    want = ts[0].dtype
    for t in ts:
        if t is not None and t.dtype is not want:
            raise RuntimeError(f"the operands must all be fp16 or all bf16; got {want} and {t.dtype}")
    if want not in _DTYPES:
        raise RuntimeError(f"the operands must be fp16 or bf16; got {want}")
    return _DTYPES[want]


def _raw_stream(t):
    """torch's current stream of t's device (which _need_cuda has found to be the current one), as a number."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _row_stride(t):
    """Row stride in elements of [T, H, D] rows that can be used in place (heads side by side, rows
    apart by a multiple of 16 bytes that holds them all, 16-byte aligned); 0 if they cannot."""
    T, H, D = t.shape
    s = t.stride()
    if (s[2] != 1 and D > 1) or (s[1] != D and H > 1) or t.data_ptr() & 15:
        return 0
    if T <= 1:
        return H * D
    return s[0] if s[0] >= H * D and not s[0] & 7 else 0


def _rows(t):
    """(t, its row stride), or a copy of it where it cannot be read in place."""
    s = _row_stride(t)
    return (t, s) if s else (t.clone(memory_format=torch.contiguous_format), t.shape[1] * t.shape[2])


def _solid(t):
    """Contiguous and 16-byte aligned (a copy where it is not)."""
    if t is None or (t.is_contiguous() and not t.data_ptr() & 15):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _span(t):
    """(first byte, row pitch in bytes, bytes of a row, rows) of a tensor whose rows are solid."""
    row = t[0].numel() * t.element_size()
    pitch = t.stride(0) * t.element_size() if t.shape[0] > 1 else row
    return t.data_ptr(), pitch, row, t.shape[0]


def _overlap(a, b):
    """Whether the bytes of two tensors with solid rows can meet.  Column blocks of one matrix
    interleave without meeting."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (pa, sa, wa, na), (pb, sb, wb, nb) = _span(a), _span(b)
    if pa + (na - 1) * sa + wa <= pb or pb + (nb - 1) * sb + wb <= pa:
        return False
    if sa == sb:
        d = (pb - pa) % sa                                    # b's rows begin d bytes into a's pitch
        return d < wa or d + wb > sa
    return True


def _check_output(out, shape, dtype, inputs, in_place_of=None):
    """`out` has the shape and type, can be written in place and is apart from the inputs; it may be
    `in_place_of` itself."""
    if out.shape != shape or out.dtype != dtype:
        raise RuntimeError(f"out must be {tuple(shape)} {dtype}; got {tuple(out.shape)} {out.dtype}")
    if not (_row_stride(out) if out.dim() == 3 else out.is_contiguous() and not out.data_ptr() & 15):
        raise RuntimeError("out must be written in place: solid rows, 16-byte aligned, strides in multiples of 8")
    for t in inputs:
        if _overlap(out, t):
            raise RuntimeError("out overlaps an input")
    t = in_place_of
    if t is not None and _overlap(out, t) and (out.data_ptr() != t.data_ptr() or _row_stride(out) != _row_stride(t)):
        raise RuntimeError("out overlaps an input")


def packed_attention(q, k, v, cu_seqlens, causal=False, scale=None, out=None):
    """Attention over packed sequences: q [T, H, D], k and v [T, KV, D] (fp16 or bf16; views of one
    projection are read in place), sequence b in rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 (int32
    [B + 1], ascending) -> out [T, H, D].  Head h reads key head h // (H // KV); causal: a row sees
    its sequence up to itself.  scale defaults to D ** -0.5.  Rows outside every sequence are not
    written (undefined in a new `out`).  D a multiple of 8 up to 128.  A bad table raises the
    device error flag (6) and leaves rows unwritten.  Not differentiable."""
    if out is None:
        r = (_bound or _bind()).packed_attention(q, k, v, cu_seqlens, causal, scale)
        if r is not None:
            return _lib.check(r) if type(r) is int else r
    _need_cuda(q, k, v, cu_seqlens, out)
    dt = _dtype16(q, k, v)
    shape, kshape = q.shape, k.shape
    if len(shape) != 3 or len(kshape) != 3 or kshape != v.shape or shape[0] != kshape[0] or shape[2] != kshape[2]:
        raise RuntimeError(f"q [T, H, D], k and v [T, KV, D] wanted; got {tuple(shape)}, {tuple(kshape)}, "
                           f"{tuple(v.shape)}")
    if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < 1 or cu_seqlens.dtype not in (torch.int32, torch.int64):
        raise RuntimeError("cu_seqlens must be int32 [B + 1]")
    if cu_seqlens.dtype is not torch.int32 or not cu_seqlens.is_contiguous():
        cu_seqlens = cu_seqlens.clamp(-1, 2 ** 31 - 1).to(torch.int32).contiguous()
    (q, qs), (k, ks), (v, vs) = _rows(q), _rows(k), _rows(v)
    T, H, D = shape
    if out is None:
        out, os = torch.empty_like(q, memory_format=torch.contiguous_format), H * D
    else:
        _check_output(out, shape, q.dtype, (q, k, v))
        os = _row_stride(out)
    rc = _lib.lib().ragrt_enc_packed_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_seqlens.data_ptr(), out.data_ptr(), T, cu_seqlens.shape[0] - 1, H,
        kshape[1], D, qs, ks, vs, os, D ** -0.5 if scale is None else scale, bool(causal), dt, _raw_stream(q))
    if rc:
        _lib.check(rc)
    return out


def qk_norm_rope(q, k, cos, sin, positions, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, q_out=None,
                 k_out=None):
    """RMS norm of each query and key head (skipped where its weight is None), then the rotation by
    cos / sin [max_pos, R / 2] f32 at positions [T] (int32 or int64) of each head's first R values:
    pairs (i, i + R / 2), or neighbours with `interleaved`.  q [T, H, D], k [T, KV, D] fp16 or bf16 ->
    (q_out, k_out), which may be q and k themselves.  D a multiple of 8 in [16, 256], R a multiple
    of 16.  A position outside the table reads its row 0 and raises the device error flag (5).  Not
    differentiable."""
    if q_out is None and k_out is None:
        r = (_bound or _bind()).qk_norm_rope(q, k, cos, sin, positions, q_weight, k_weight, eps, interleaved)
        if r is not None:
            return _lib.check(r) if type(r) is int else r
    _need_cuda(q, k, cos, sin, positions, q_weight, k_weight, q_out, k_out)
    dt = _dtype16(q, k, q_weight, k_weight)
    shape, kshape = q.shape, k.shape
    if len(shape) != 3 or len(kshape) != 3 or shape[0] != kshape[0] or shape[2] != kshape[2]:
        raise RuntimeError(f"q [T, H, D] and k [T, KV, D] wanted; got {tuple(shape)}, {tuple(kshape)}")
    T, H, D = shape
    KV = kshape[1]
    if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype is not torch.float32 or sin.dtype is not torch.float32:
        raise RuntimeError("cos and sin must be f32 [max_pos, R / 2]")
    if positions.shape != (T,) or positions.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"positions must be int32 or int64 [{T}]")
    for w in (q_weight, k_weight):
        if w is not None and w.shape != (D,):
            raise RuntimeError(f"a norm weight must be [{D}]; got {tuple(w.shape)}")
    (q, qs), (k, ks) = _rows(q), _rows(k)
    cos, sin, qw, kw, pos = _solid(cos), _solid(sin), _solid(q_weight), _solid(k_weight), positions.contiguous()
    if q_out is None:
        q_out, qos = torch.empty_like(q, memory_format=torch.contiguous_format), H * D
    else:
        _check_output(q_out, shape, q.dtype, (k,), in_place_of=q)
        qos = _row_stride(q_out)
    if k_out is None:
        k_out, kos = torch.empty_like(k, memory_format=torch.contiguous_format), KV * D
    else:
        _check_output(k_out, kshape, k.dtype, (q, q_out), in_place_of=k)
        kos = _row_stride(k_out)
    rc = _lib.lib().ragrt_enc_qk_norm_rope(
        q.data_ptr(), k.data_ptr(), qw if qw is None else qw.data_ptr(), kw if kw is None else kw.data_ptr(),
        cos.data_ptr(), sin.data_ptr(), pos.data_ptr(), pos.element_size(), q_out.data_ptr(), k_out.data_ptr(), T, H,
        KV, D, 2 * cos.shape[1], cos.shape[0], qs, ks, qos, kos, eps, bool(interleaved), dt, _raw_stream(q))
    if rc:
        _lib.check(rc)
    return q_out, k_out


def _ffn_args(x, w_gate, w_up, act):
    if act not in _ACTS:
        raise RuntimeError(f"unknown activation {act!r}: one of {sorted(_ACTS)}")
    shape, wshape = x.shape, w_gate.shape
    if len(shape) != 2 or len(wshape) != 2 or wshape != w_up.shape or wshape[1] != shape[1]:
        raise RuntimeError(f"x [M, K], w_gate and w_up [F, K] wanted; got {tuple(shape)}, {tuple(wshape)}, "
                           f"{tuple(w_up.shape)}")
    return shape[0], wshape[0], shape[1]


def gated_ffn(x, w_gate, w_up, act="silu", keep=False, out=None):
    """h [M, F] = act(x w_gate^T) * (x w_up^T) in one kernel: x [M, K], weights [F, K] (the halves of
    a stacked [2 F, K] matrix are read in place), fp16 or bf16, F and K multiples of 8; act "silu",
    "gelu" (erf form) or "gelu_tanh".  keep=True returns (h, gate, up) with the two products in
    fp32, which gated_ffn_backward wants.  Not tracked by autograd."""
    if out is None and act in _ACTS:
        r = (_bound or _bind()).gated_ffn(x, w_gate, w_up, _ACTS[act], keep)
        if r is not None:
            return _lib.check(r) if type(r) is int else r
    _need_cuda(x, w_gate, w_up, out)
    dt = _dtype16(x, w_gate, w_up)
    M, F, K = _ffn_args(x, w_gate, w_up, act)
    x, wg, wu = _solid(x), _solid(w_gate), _solid(w_up)
    if out is None:
        out = x.new_empty((M, F))
    else:
        _check_output(out, (M, F), x.dtype, (x, wg, wu))
    gate = up = None
    if keep:
        gate, up = torch.empty_like(out, dtype=torch.float32), torch.empty_like(out, dtype=torch.float32)
    rc = _lib.lib().ragrt_enc_gated_ffn(
        x.data_ptr(), wg.data_ptr(), wu.data_ptr(), out.data_ptr(), gate.data_ptr() if keep else None,
        up.data_ptr() if keep else None, M, F, K, _ACTS[act], dt, _raw_stream(x))
    if rc:
        _lib.check(rc)
    return (out, gate, up) if keep else out


def gated_ffn_backward(dh, x, w_gate, w_up, gate, up, act="silu", need_dx=True, need_dw=True):
    """Gradients of gated_ffn from dh [M, F] and the kept gate and up: (dx [M, K], dw_gate [F, K],
    dw_up [F, K]) in the inputs' type, None for what is not needed.  Sums run in a fixed order."""
    if act in _ACTS:
        r = (_bound or _bind()).gated_ffn_backward(dh, x, w_gate, w_up, gate, up, _ACTS[act], need_dx, need_dw)
        if r is not None:
            return _lib.check(r) if type(r) is int else r
    _need_cuda(dh, x, w_gate, w_up, gate, up)
    dt = _dtype16(dh, x, w_gate, w_up)
    if gate.dtype is not torch.float32 or up.dtype is not torch.float32:
        raise RuntimeError(f"gate and up must be fp32, as gated_ffn keeps them; got {gate.dtype} and {up.dtype}")
    M, F, K = _ffn_args(x, w_gate, w_up, act)
    if dh.shape != (M, F) or gate.shape != (M, F) or up.shape != (M, F):
        raise RuntimeError(f"dh, gate and up must be {(M, F)}; got {tuple(dh.shape)}, {tuple(gate.shape)}, "
                           f"{tuple(up.shape)}")
    dh, x, wg, wu, gate, up = (_solid(t) for t in (dh, x, w_gate, w_up, gate, up))
    dgate, dup = torch.empty_like(dh), torch.empty_like(dh)
    dx = torch.empty_like(x) if need_dx else None
    dwg, dwu = (torch.empty_like(wg), torch.empty_like(wu)) if need_dw else (None, None)
    nbytes = _lib.lib().ragrt_enc_gated_ffn_workspace(M, F, K, bool(need_dx), bool(need_dw))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    _lib.check(_lib.lib().ragrt_enc_gated_ffn_backward(
        dh.data_ptr(), x.data_ptr(), wg.data_ptr(), wu.data_ptr(), gate.data_ptr(), up.data_ptr(), dgate.data_ptr(),
        dup.data_ptr(), dx.data_ptr() if need_dx else None, dwg.data_ptr() if need_dw else None,
        dwu.data_ptr() if need_dw else None, M, F, K, _ACTS[act], dt, ws.data_ptr(), ws.numel(), _raw_stream(x)))
    return dx, dwg, dwu


class FastQueryEncoder:
    """encode(text) -> ([32, 128] fp16, ntok); encode_batch(texts) -> ([B, 32, 128] fp16, ntoks)."""

    def __init__(self, checkpoint=None, device="cuda", use_graphs=True, weights=None, tokenizer=None):
        self.tok = tokenizer if tokenizer is not None else getattr(checkpoint, "query_tokenizer", None)
        if weights is None:
            bert, linear = bert_and_linear(checkpoint)
            weights = flat_weights(bert, linear, device=device)
        self.W = weights
        self.device, self.use_graphs = device, use_graphs
        self.graphs = {}

    def tokenize(self, texts):
        if self.tok is None:
            raise RuntimeError("no query tokenizer: pass token ids to encode_ids")
        return self.tok.tensorize(list(texts))

    def _graph(self, B, L):
        key = (B, L)
        if key not in self.graphs:
            ids = torch.zeros(B, L, dtype=torch.int64, device=self.device)
            mask = torch.ones(B, L, dtype=torch.int64, device=self.device)
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s), torch.no_grad():
                for _ in range(2):
                    flat_forward(self.W, ids, mask)
            torch.cuda.current_stream().wait_stream(s)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g), torch.no_grad():
                out = flat_forward(self.W, ids, mask)
            self.graphs[key] = (g, ids, mask, out)
        return self.graphs[key]

    @torch.no_grad()
    def encode_ids(self, ids, mask):
        """Token ids and attention mask [B, L] (host or device) -> [B, L, 128] fp16 on the device."""
        if not self.use_graphs:
            return flat_forward(self.W, ids.to(self.device), mask.to(self.device))
        g, gi, gm, out = self._graph(*ids.shape)
        gi.copy_(ids, non_blocking=True)
        gm.copy_(mask, non_blocking=True)
        g.replay()
        return out.clone()

    @torch.no_grad()
    def encode_batch(self, texts):
        ids, mask = self.tokenize(texts)
        ntoks = mask.sum(1).tolist()
        return self.encode_ids(ids, mask), ntoks

    def encode(self, text):
        Q, ntoks = self.encode_batch([text])
        return Q[0].contiguous(), int(ntoks[0])
