"""Host-side operator surface over the C ABI (device memory via torch).

MoeLayer owns one layer's device weights in the layout include/ainfer_moe.h
documents; forward/route/dispatch/block_forward enqueue on a HIP stream and
return immediately, like the C entry points they wrap.  Every call goes to
libainfer_moe.so; there is no other implementation behind these names.
"""
import contextlib
import ctypes as C

import numpy as np
import torch

from . import _lib as L
from .synthetic import MoeConfig, tensor_seed, layer_seed, input_seed, zipf_bias


def _ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else C.c_void_p(0)


def _stream(stream):
    if stream is None:
        stream = torch.cuda.current_stream()
    return C.c_void_p(stream.cuda_stream)


def _on(stream):
    """The stream as torch's current one (buffers allocated under it are its
    own); nothing to do for None."""
    return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)


def fill_(kind: int, seed: int, std: float, t: torch.Tensor, stream=None):
    """Fill a device tensor with the counter-based synthetic generator."""
    n = t.numel() * t.element_size() if kind == L.FILL_BYTES else t.numel()
    L.check(L.lib().ainfer_moe_fill(kind, C.c_uint64(seed), C.c_float(std), n, _ptr(t),
                                    _stream(stream)))
    return t


class MoeLayer:
    """One INT4 MoE layer resident in HBM (synthetic seeded weights)."""

    def __init__(self, cfg: MoeConfig, layer: int = 0, device="cuda",
                 scale_dtype: int = L.SCALE_FP16, stream=None,
                 precision: int = L.PRECISION_W4A16):
        self.cfg, self.layer, self.device = cfg, layer, device
        H, E, I, Is = cfg.hidden, cfg.n_experts, cfg.inter, cfg.shared_inter
        self.shape = L.Shape(H, E, cfg.top_k, I, Is, 128, scale_dtype, precision)
        L.check(L.lib().ainfer_moe_validate(C.byref(self.shape)))
        ls = layer_seed(cfg.seed, layer)
        sdt = torch.float16 if scale_dtype == L.SCALE_FP16 else torch.bfloat16
        skind = L.FILL_FP16_ABSNORMAL if scale_dtype == L.SCALE_FP16 else L.FILL_BF16_ABSNORMAL
        u8 = dict(dtype=torch.uint8, device=device)

        def packed(name, rows, K, n_mat=1):
            return fill_(L.FILL_BYTES, tensor_seed(ls, name), 0.0,
                         torch.empty(n_mat * rows * K // 2, **u8), stream)

        def scales(name, rows, K, n_mat=1):
            return fill_(skind, tensor_seed(ls, name), cfg.scale_std,
                         torch.empty(n_mat * rows * K // 128, dtype=sdt, device=device), stream)

        t = {}
        t["router_w"] = fill_(L.FILL_BF16_NORMAL, tensor_seed(ls, "router_w"), cfg.weight_std,
                              torch.empty(E * H, dtype=torch.bfloat16, device=device), stream)
        t["shared_gate_w"] = (fill_(L.FILL_BF16_NORMAL, tensor_seed(ls, "shared_gate_w"),
                                    cfg.weight_std,
                                    torch.empty(H, dtype=torch.bfloat16, device=device), stream)
                              if cfg.shared_gate and Is > 0 else None)
        t["router_bias"] = (torch.from_numpy(zipf_bias(cfg, layer)).to(device)
                            if cfg.zipf > 0 else None)
        t["w_gate"], t["s_gate"] = packed("w_gate", I, H, E), scales("s_gate", I, H, E)
        t["w_up"], t["s_up"] = packed("w_up", I, H, E), scales("s_up", I, H, E)
        t["w_down"], t["s_down"] = packed("w_down", H, I, E), scales("s_down", H, I, E)
        if Is > 0:
            t["ws_gate"], t["ss_gate"] = packed("ws_gate", Is, H), scales("ss_gate", Is, H)
            t["ws_up"], t["ss_up"] = packed("ws_up", Is, H), scales("ss_up", Is, H)
            t["ws_down"], t["ss_down"] = packed("ws_down", H, Is), scales("ss_down", H, Is)
        self.t = t
        self.weights = L.Weights(*[_ptr(t.get(n)) for n, _ in L.Weights._fields_])

    def set_tensor(self, name: str, t):
        """Replace one device tensor (same layout) and refresh the C struct."""
        self.t[name] = t
        self.weights = L.Weights(*[_ptr(self.t.get(n)) for n, _ in L.Weights._fields_])

    def workspace(self, max_tokens: int) -> torch.Tensor:
        n = L.lib().ainfer_moe_workspace_bytes(C.byref(self.shape), max_tokens)
        if n == 0:
            raise L.MoeError("invalid shape or token count for workspace")
        ws = torch.empty(n + 256, dtype=torch.uint8, device=self.device)
        off = (-ws.data_ptr()) % 256
        ws = ws[off:off + n]
        L.check(L.lib().ainfer_moe_workspace_init(C.byref(self.shape), _ptr(ws), n, _stream(None)))
        return ws

    def workspace_check(self, ws, stream=None) -> int:
        """Status of the workspace's synchronisation words (OK when all zero)."""
        return L.lib().ainfer_moe_workspace_check(C.byref(self.shape), _ptr(ws), ws.numel(),
                                                  _stream(stream))

    def forward(self, x, y, ws, stream=None):
        T = x.shape[0]
        return L.check(L.lib().ainfer_moe_forward(
            C.byref(self.shape), C.byref(self.weights), _ptr(x), _ptr(y), T, _ptr(ws),
            ws.numel(), _stream(stream)))

    def block_forward(self, resid_in, resid_out, ws, norm_w=None, norm_mode=L.NORM_PLAIN,
                      eps=1e-6, stream=None):
        T = resid_in.shape[0]
        return L.check(L.lib().ainfer_moe_block_forward(
            C.byref(self.shape), C.byref(self.weights), _ptr(norm_w), norm_mode, eps,
            _ptr(resid_in), _ptr(resid_out), T, _ptr(ws), ws.numel(), _stream(stream)))

    def block_forward_noalloc(self, resid_in, resid_out, norm_w=None, norm_mode=L.NORM_PLAIN,
                              eps=1e-6, stream=None):
        """block_forward on the library's static per-GPU scratch (no workspace)."""
        T = resid_in.shape[0]
        return L.check(L.lib().ainfer_moe_block_forward_noalloc(
            C.byref(self.shape), C.byref(self.weights), _ptr(norm_w), norm_mode, eps,
            _ptr(resid_in), _ptr(resid_out), T, _stream(stream)))

    def route(self, x, ws, want_logits=False, stream=None):
        T, E, k = x.shape[0], self.shape.n_experts, self.shape.top_k
        dev = self.device
        idx = torch.empty(T, k, dtype=torch.int32, device=dev)
        w = torch.empty(T, k, dtype=torch.float32, device=dev)
        sg = torch.empty(T, dtype=torch.float32, device=dev)
        lg = torch.empty(T, E, dtype=torch.float32, device=dev) if want_logits else None
        L.check(L.lib().ainfer_moe_route(C.byref(self.shape), C.byref(self.weights), _ptr(x), T,
                                         _ptr(idx), _ptr(w), _ptr(sg), _ptr(lg), _ptr(ws),
                                         ws.numel(), _stream(stream)))
        return idx, w, sg, lg

    def experts(self, x, idx, ws, stream=None):
        """Expert rows in slot order: [T * k + T][H] bf16 (row t * k + j =
        expert idx[t][j] on token t, row T * k + t = the shared expert)."""
        T, k, H = x.shape[0], self.shape.top_k, self.shape.hidden
        o = torch.empty(T * k + T, H, dtype=torch.bfloat16, device=self.device)
        L.check(L.lib().ainfer_moe_experts(C.byref(self.shape), C.byref(self.weights), _ptr(x),
                                           _ptr(idx), T, _ptr(o), _ptr(ws), ws.numel(),
                                           _stream(stream)))
        return o

    def combine(self, o, w, sg, y, resid=None, stream=None):
        T = y.shape[0]
        L.check(L.lib().ainfer_moe_combine(C.byref(self.shape), _ptr(o), _ptr(w), _ptr(sg),
                                           _ptr(resid), _ptr(y), T, _stream(stream)))
        return y

    def forward_scored(self, x, y, ws, routing, bias=None, resid=None, shared=None, stream=None,
                       shared_tokens=None):
        """forward with scored routing: the layer's router logits (its
        router_bias, where it has one, is part of them) -> route_scored(routing,
        logits, bias) -> experts -> combine, in steps of CHUNK_TOKENS (ws: for
        that many tokens, or T where it is less).  W4A16 layers only, as
        ainfer_moe_experts.  shared: [T][H] bf16 rows that take the place of the
        shared expert's (for example shared_adapted's, whose activations are
        int8); shared_tokens: [T] bool, the tokens they do so for (token_adapter >= 0,
        say, so that a token without an adapter has the layer's own W4A16 row
        whoever shares its batch), None for all."""
        if self.shape.precision != L.PRECISION_W4A16:
            raise L.MoeError("forward_scored: a W4A16 layer (the expert stage has no W4A8 form)")
        if (routing.n_experts, routing.top_k) != (self.shape.n_experts, self.shape.top_k):
            raise L.MoeError("routing: the layer's n_experts and top_k")
        T, H, dev = x.shape[0], self.shape.hidden, x.get_device()
        for t in (x, y, resid, shared):
            if t is not None and not (t.shape == (T, H) and t.dtype == torch.bfloat16
                                      and t.is_contiguous() and t.get_device() == dev >= 0):
                raise L.MoeError("x, y, resid and shared: contiguous [T][H] bf16 on one device")
        if ws.get_device() != dev:
            raise L.MoeError("ws: on the inputs' device")
        if bias is not None:
            _vector(bias, "bias", torch.float32, routing.n_experts, dev)
        L.check(L.lib().ainfer_moe_route_scored(C.byref(routing), None, L.ACT_F32, 0, None, 0, None,
                                                None, None))  # no tokens: routing's own checks
        if shared is not None and self.shape.shared_inter == 0:
            raise L.MoeError("shared: the layer has no shared expert")
        if shared_tokens is not None:
            if shared is None:
                raise L.MoeError("shared_tokens: the tokens of shared")
            _vector(shared_tokens, "shared_tokens", torch.bool, T, dev)
        with torch.cuda.device(dev), _on(stream):
            for t in range(0, T, L.CHUNK_TOKENS):
                c = slice(t, t + L.CHUNK_TOKENS)
                idx, w, sg, logits = self.route(x[c], ws, want_logits=True)
                route_scored(routing, logits, bias, out=(idx, w))
                o = self.experts(x[c], idx, ws)
                if shared_tokens is not None:
                    own = o[idx.numel():]
                    torch.where(shared_tokens[c, None], shared[c], own, out=own)
                elif shared is not None:
                    o[idx.numel():].copy_(shared[c])
                self.combine(o, w, sg, y[c], resid[c] if resid is not None else None)
        return y

    def shared_adapted(self, x, token_adapter, gate_up, down, lora_ws, stream=None):
        """The shared expert's rows [T][H] (bf16) with each token's adapters on
        its three projections: x quantised to int8 groups, gate and up as
        ainfer_moe_int4_gemv_i8, their adapters, SiLU-mul, the same for down.
        That is W4A8 arithmetic whatever the layer's precision: rows of a W4A16 layer
        differ from its own shared expert's by the rounding of x and act to int8,
        without an adapter too (forward_scored's shared_tokens keeps the
        layer's own for those).
        gate_up (two projections, x bf16, y fp32) and down (x and y fp32):
        LoraAdapters or None; lora_ws: a workspace large enough for both."""
        sh, wt = self.shape, self.weights
        H, Is = sh.hidden, sh.shared_inter
        if Is == 0 or x.shape[1] != H:
            raise L.MoeError("a layer with a shared expert, x of its hidden size")
        with _on(stream):
            q, sq = act_quant_i8(x)
            gate = int4_gemv_i8(wt.ws_gate, wt.ss_gate, sh.scale_dtype, q, sq, Is)
            up = int4_gemv_i8(wt.ws_up, wt.ss_up, sh.scale_dtype, q, sq, Is)
            if gate_up is not None:
                gate_up.apply(x, token_adapter, [gate, up], lora_ws)
            act = silu_mul(gate, up, gate)
            q, sq = act_quant_i8(act)
            out = int4_gemv_i8(wt.ws_down, wt.ss_down, sh.scale_dtype, q, sq, H)
            if down is not None:
                down.apply(act, token_adapter, [out], lora_ws)
            return out.to(torch.bfloat16)

    def dispatch(self, idx, ws, stream=None):
        T, E, k = idx.shape[0], self.shape.n_experts, self.shape.top_k
        dev = self.device
        counts = torch.empty(E, dtype=torch.int32, device=dev)
        offsets = torch.empty(E + 1, dtype=torch.int32, device=dev)
        perm = torch.empty(max(T * k, 1), dtype=torch.int32, device=dev)
        inv = torch.empty(max(T * k, 1), dtype=torch.int32, device=dev)
        L.check(L.lib().ainfer_moe_dispatch(C.byref(self.shape), _ptr(idx), T, _ptr(counts),
                                            _ptr(offsets), _ptr(perm), _ptr(inv), _ptr(ws),
                                            ws.numel(), _stream(stream)))
        return counts, offsets, perm[:T * k], inv[:T * k]


def load_binfer_layer(bf, layer, device="cuda"):
    """Layer `layer` of an opened BinferFile, copied into a device arena: a
    MoeLayer whose weights are the file's (no synthetic fill); its norm
    weight (or None) is returned beside it."""
    shape, n_layers, eps = bf.moe_info()
    nbytes = bf.layer_bytes(layer)
    arena = torch.empty(nbytes + 256, dtype=torch.uint8, device=device)
    off = (-arena.data_ptr()) % 256
    arena = arena[off:off + nbytes]
    w = L.Weights()
    nw = C.c_void_p()
    L.check(L.lib().ainfer_binfer_load_moe_layer(bf.h, layer, _ptr(arena), nbytes, C.byref(w),
                                                 C.byref(nw), _stream(None)))
    ly = MoeLayer.__new__(MoeLayer)
    ly.cfg = None
    ly.device = device
    ly.shape = shape
    ly.weights = w
    ly.t = {"arena": arena}
    norm = None
    if nw.value:
        # a view of the arena at the norm weight's offset
        norm = arena[nw.value - arena.data_ptr():][:shape.hidden * 2].view(torch.bfloat16)
    return ly, norm


def with_precision(layer, precision):
    """The same resident layer (shared weights) run in another precision."""
    twin = MoeLayer.__new__(MoeLayer)
    twin.__dict__.update(layer.__dict__)
    twin.shape = L.Shape.from_buffer_copy(layer.shape)
    twin.shape.precision = precision
    L.check(L.lib().ainfer_moe_validate(C.byref(twin.shape)))
    return twin


class MoeStack:
    """L decoder-block MLP halves as one call (ainfer_moe_stack_forward: the
    layers' kernels replayed, each layer's combine computing the next layer's
    RMSNorm; any T), or as one persistent launch
    (ainfer_moe_stack_forward_persistent, T <= 4).  The layers' weights and
    per-layer RMSNorm weights go into a device table once
    (ainfer_moe_stack_prepare)."""

    def __init__(self, layers, norm_ws=None, device="cuda"):
        assert layers, "a stack needs at least one layer"
        self.layers = list(layers)
        self.shape = self.layers[0].shape
        n = len(self.layers)
        lib = L.lib()
        self.table = torch.empty(lib.ainfer_moe_stack_table_bytes(n), dtype=torch.uint8,
                                 device=device)
        arr = (L.Weights * n)(*[ly.weights for ly in self.layers])
        self.norm_ws = list(norm_ws) if norm_ws is not None else None
        nw = None
        if self.norm_ws is not None:
            assert len(self.norm_ws) == n
            nw = (C.c_void_p * n)(*[_ptr(w) for w in self.norm_ws])
        L.check(lib.ainfer_moe_stack_prepare(C.byref(self.shape), arr, nw, n,
                                             _ptr(self.table), self.table.numel(), None))

    def workspace(self, max_tokens: int) -> torch.Tensor:
        lib = L.lib()
        n = lib.ainfer_moe_stack_workspace_bytes(C.byref(self.shape), max_tokens, len(self.layers))
        if n == 0:
            raise L.MoeError("invalid shape or token count for a stack workspace")
        ws = torch.empty(n + 256, dtype=torch.uint8, device=self.table.device)
        off = (-ws.data_ptr()) % 256
        ws = ws[off:off + n]
        L.check(lib.ainfer_moe_workspace_init(C.byref(self.shape), _ptr(ws), n, _stream(None)))
        return ws

    def forward(self, resid_in, resid_out, ws, norm_mode=L.NORM_PLAIN, eps=1e-6, stream=None,
                persistent=False):
        T = resid_in.shape[0]
        fn = (L.lib().ainfer_moe_stack_forward_persistent if persistent
              else L.lib().ainfer_moe_stack_forward)
        return L.check(fn(
            C.byref(self.shape), _ptr(self.table), len(self.layers), norm_mode, eps,
            _ptr(resid_in), _ptr(resid_out), T, _ptr(ws), ws.numel(), _stream(stream)))


def make_input(cfg: MoeConfig, T: int, tag: int = 0, device="cuda", stream=None):
    """x[T][H] bf16 ~ N(0, 1) (standardised Irwin-Hall), seeded by (cfg.seed, tag)."""
    x = torch.empty(T, cfg.hidden, dtype=torch.bfloat16, device=device)
    return fill_(L.FILL_BF16_NORMAL, input_seed(cfg.seed, tag), 1.0, x, stream)


def rmsnorm(x, y, w=None, mode=L.NORM_PLAIN, eps=1e-6, stream=None):
    T, H = x.shape
    return L.check(L.lib().ainfer_moe_rmsnorm(_ptr(x), _ptr(w), mode, eps, _ptr(y), T, H,
                                              _stream(stream)))


# ---- the operators around the expert stage -----------------------------------
# These calls are short (a kernel takes a few microseconds), so the checks below
# read each tensor attribute once and pass plain integers to the library.
_ACT = {torch.float32: L.ACT_F32, torch.bfloat16: L.ACT_BF16}


def _rows(t, name, cols=None):
    """A device matrix of fp32 or bf16 rows, each contiguous: (dtype, device,
    rows, columns, pitch)."""
    dt, dev = _ACT.get(t.dtype), t.get_device()
    if dt is None or dev < 0 or t.dim() != 2:
        raise L.MoeError(f"{name}: a device matrix of fp32 or bf16 rows")
    n, m = t.shape
    ld, one = t.stride()
    if (cols is not None and m != cols) or (one != 1 and m != 1):
        raise L.MoeError(f"{name}: contiguous rows" + (f" of {cols} columns" if cols else ""))
    return dt, dev, n, m, (ld if n > 1 else m)  # a single row has no pitch


def _vector(t, name, dtype, n, dev):
    if t.dtype != dtype or t.shape != (n,) or t.get_device() != dev or not t.is_contiguous():
        raise L.MoeError(f"{name}: {n} contiguous {dtype} values on the inputs' device")


def _call(fn, dev, stream, *args):
    """fn(*args, stream) on the device the tensors are on; its current stream
    when none is given."""
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return _enqueue(fn, dev, stream, args)
    return _enqueue(fn, dev, stream, args)


def _enqueue(fn, dev, stream, args):
    raw = torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream
    rc = fn(*args, raw)
    if rc:
        L.check(rc)


def route_scored(routing, logits, bias=None, out=None, stream=None):
    """Scored routing of logits [T][E] (ainfer_moe_route_scored; routing: an
    L.Routing): (topk_idx [T][k] int32, topk_w [T][k] fp32), as MoeLayer.dispatch,
    experts and combine take them.  out: the two tensors to write."""
    dt, dev, T, E, ld = _rows(logits, "logits", routing.n_experts)
    k = routing.top_k
    if bias is not None:
        _vector(bias, "bias", torch.float32, E, dev)
    if out is None:
        with _on(stream):
            idx = torch.empty(T, k, dtype=torch.int32, device=logits.device)
            w = torch.empty(T, k, dtype=torch.float32, device=logits.device)
    else:
        idx, w = out
        if not (idx.dtype == torch.int32 and w.dtype == torch.float32
                and idx.shape == w.shape == (T, k) and idx.get_device() == dev == w.get_device()
                and idx.is_contiguous() and w.is_contiguous()):
            raise L.MoeError("out: (idx int32, w fp32), [T][k] contiguous on the logits' device")
    _call(L.lib().ainfer_moe_route_scored, dev, stream, C.byref(routing), logits.data_ptr(), dt,
          ld, bias.data_ptr() if bias is not None else None, T, idx.data_ptr(), w.data_ptr())
    return idx, w


def act_quant_i8(x, stream=None):
    """int8 codes [T][K] and group scales [T][K / 128] of contiguous x
    (ainfer_moe_act_quant_i8)."""
    dt, dev, T, K, ld = _rows(x, "x")
    if ld != K:
        raise L.MoeError("x: contiguous")
    with _on(stream):
        q = torch.empty(T, K, dtype=torch.int8, device=x.device)
        sq = torch.empty(T, K // 128, dtype=torch.float32, device=x.device)
    _call(L.lib().ainfer_moe_act_quant_i8, dev, stream, x.data_ptr(), dt, T, K, q.data_ptr(),
          sq.data_ptr())
    return q, sq


def int4_gemv_i8(packed, scales, scale_dtype, q, sq, rows, stream=None):
    """y [T][rows] fp32 of an INT4 matrix (device addresses of its nibbles and
    scales) and act_quant_i8's codes (ainfer_moe_int4_gemv_i8)."""
    T, K = q.shape
    dev = q.get_device()
    _vector(sq.view(-1), "sq", torch.float32, T * (K // 128), dev)
    if q.dtype != torch.int8 or not q.is_contiguous() or dev < 0:
        raise L.MoeError("q: contiguous int8 rows on a device")
    with _on(stream):
        y = torch.empty(T, rows, dtype=torch.float32, device=q.device)
    _call(L.lib().ainfer_moe_int4_gemv_i8, dev, stream, packed, scales, scale_dtype, q.data_ptr(),
          sq.data_ptr(), rows, K, T, y.data_ptr())
    return y


def silu_mul(gate, up, act, stream=None):
    """act = gate / (1 + exp(-gate)) * up over rows of any pitch
    (ainfer_moe_silu_mul); act may be gate or up."""
    dt, dev, T, n, gld = _rows(gate, "gate")
    udt, udev, uT, _, uld = _rows(up, "up", n)
    adt, adev, aT, _, ald = _rows(act, "act", n)
    if not (udt == dt and uT == T == aT and udev == dev == adev):
        raise L.MoeError("gate, up and act: one shape and device, gate and up one type")
    _call(L.lib().ainfer_moe_silu_mul, dev, stream, gate.data_ptr(), gld, up.data_ptr(), uld, dt,
          T, n, act.data_ptr(), ald, adt)
    return act


class LoraAdapters:
    """The adapters of up to LORA_MAX_PROJ projections of one input, resident
    on one device: a[p] [N][R][K] and b[p] [N][M_p][R] bf16, optional ranks
    ([N] int32, the rows of each adapter in use) and scales ([N] fp32)."""

    def __init__(self, a, b, ranks=None, scales=None, x_dtype=torch.bfloat16,
                 y_dtype=torch.bfloat16):
        a, b = list(a), list(b)
        if not 1 <= len(a) == len(b) <= L.LORA_MAX_PROJ:
            raise L.MoeError("one a and one b for each of up to "
                             f"{L.LORA_MAX_PROJ} projections")
        if x_dtype not in _ACT or y_dtype not in _ACT:
            raise L.MoeError("x and y: fp32 or bf16")
        dev = a[0].get_device()
        for t in a + b:
            if not (t.dtype == torch.bfloat16 and t.get_device() == dev >= 0
                    and t.is_contiguous() and t.dim() == 3):
                raise L.MoeError("a and b: contiguous [N][R][K] and [N][M][R] bf16 on one device")
        N, R, K = a[0].shape
        for ta, tb in zip(a, b):
            if ta.shape != (N, R, K) or tb.shape[0] != N or tb.shape[2] != R:
                raise L.MoeError("a [N][R][K] and b [N][M][R] of one N, R and K")
        if ranks is not None:
            _vector(ranks, "ranks", torch.int32, N, dev)
        if scales is not None:
            _vector(scales, "scales", torch.float32, N, dev)
        self.tensors = (a, b, ranks, scales)
        self.device, self.dev, self.x_dtype, self.y_dtype = a[0].device, dev, x_dtype, y_dtype
        self.cols, self.rows = K, [t.shape[1] for t in b]
        s = L.Lora(N, R, K, len(a), _ACT[x_dtype], _ACT[y_dtype])
        for p, (ta, tb) in enumerate(zip(a, b)):
            s.out[p], s.a[p], s.b[p] = tb.shape[1], ta.data_ptr(), tb.data_ptr()
        s.ranks = ranks.data_ptr() if ranks is not None else None
        s.scales = scales.data_ptr() if scales is not None else None
        self.struct = s
        if L.lib().ainfer_moe_lora_workspace_bytes(C.byref(s), 1) == 0:
            raise L.MoeError("adapter sizes outside the supported range")

    def workspace(self, max_tokens):
        """Scratch for calls with up to max_tokens tokens (no initialisation)."""
        n = L.lib().ainfer_moe_lora_workspace_bytes(C.byref(self.struct), max_tokens)
        if n == 0:
            raise L.MoeError("invalid token count for an adapter workspace")
        ws = torch.empty(n + 256, dtype=torch.uint8, device=self.device)
        off = (-ws.data_ptr()) % 256
        return ws[off:off + n]

    def apply(self, x, token_adapter, ys, ws, stream=None):
        """ys[p] += scale * (x a^T) b^T of each token's adapter, in place
        (ainfer_moe_lora_apply); tokens without one keep their rows."""
        dev = self.dev
        _, xdev, T, _, ld = _rows(x, "x", self.cols)
        if x.dtype != self.x_dtype or xdev != dev or ws.get_device() != dev or \
                not ws.is_contiguous():
            raise L.MoeError("x: the adapters' x type; x and the workspace on their device")
        _vector(token_adapter, "token_adapter", torch.int32, T, dev)
        if len(ys) != len(self.rows):
            raise L.MoeError("one y per projection")
        yp, yl = (C.c_void_p * len(ys))(), (C.c_int64 * len(ys))()
        for p, y in enumerate(ys):
            _, ydev, n, _, yl[p] = _rows(y, "y", self.rows[p])
            if n != T or y.dtype != self.y_dtype or ydev != dev:
                raise L.MoeError("y: a row per token, of the adapters' y type and device")
            yp[p] = y.data_ptr()
        _call(L.lib().ainfer_moe_lora_apply, dev, stream, C.byref(self.struct), x.data_ptr(), ld,
              token_adapter.data_ptr(), T, yp, yl, ws.data_ptr(), ws.nbytes)
        return ys
