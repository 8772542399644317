"""Host-side operator surface over the C ABI (device memory via torch).

MoeLayer owns one layer's device weights in the layout include/ainfer_moe.h
documents; forward/route/dispatch/block_forward enqueue on a HIP stream and
return immediately, like the C entry points they wrap.  Every call goes to
libainfer_moe.so; there is no other implementation behind these names.
"""
import contextlib
import ctypes as C
import functools

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


_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _call(fn, dev, stream, *args):
    """fn(*args, stream) on the device the tensors are on; its current stream
    when none is given."""
    if dev != _current_device():
        with torch.cuda.device(dev):
            return _call(fn, dev, stream, *args)
    rc = fn(*args, _raw_stream(dev) if stream is None else stream.cuda_stream)
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


# ---- experts in 8-bit floating point -------------------------------------------
_CODES = (torch.float8_e4m3fn, torch.uint8)


def _codes(t, name, cols=None):
    """A device matrix of e4m3 codes (as float8_e4m3fn or uint8), rows contiguous:
    (device, rows, columns, pitch)."""
    dev = t.get_device()
    if t.dtype not in _CODES or dev < 0 or t.dim() != 2:
        raise L.MoeError(f"{name}: a device matrix of float8_e4m3fn or uint8 codes")
    n, m = t.shape
    ld, one = t.stride()
    if (cols is not None and m != cols) or (one != 1 and m != 1):
        raise L.MoeError(f"{name}: contiguous rows" + (f" of {cols} columns" if cols else ""))
    return dev, n, m, (ld if n > 1 else m)


def _scales(t, name, n, cols, dev):
    if not (t.dtype == torch.float32 and t.shape == (n, -(-cols // 128))
            and t.get_device() == dev and t.is_contiguous()):
        raise L.MoeError(f"{name}: contiguous fp32 [{n}][{-(-cols // 128)}] on the rows' device")


def _live(live, dev):
    """The address of a device count of rows: the last value of an int32 vector
    (sort_rows' offsets, say)."""
    if live is None:
        return None
    if live.dtype != torch.int32 or live.dim() != 1 or live.get_device() != dev or \
            not live.is_contiguous() or live.numel() == 0:
        raise L.MoeError("live: a contiguous int32 vector on the rows' device")
    return live.data_ptr() + 4 * (live.numel() - 1)


def _kind(pow2):
    return L.FP8_SCALE_POW2 if pow2 else L.FP8_SCALE_ANY


def _new_codes(n, cols, device):
    return (torch.empty(n, cols, dtype=torch.float8_e4m3fn, device=device),
            torch.empty(n, -(-cols // 128), dtype=torch.float32, device=device))


def act_quant_fp8(x, q=None, sq=None, pow2=False, live=None, stream=None):
    """e4m3 codes [N][K] and scales [N][ceil(K / 128)] of the rows of x
    (ainfer_moe_act_quant_fp8), in q and sq where these are given.  live: an int32
    vector whose last value is how many rows to take (sort_rows' offsets)."""
    dt, dev, n, K, ld = _rows(x, "x")
    if (q is None) != (sq is None):
        raise L.MoeError("q and sq: both or neither")
    if q is None:
        with _on(stream):
            q, sq = _new_codes(n, K, x.device)
    qdev, qn, _, qld = _codes(q, "q", K)
    if qdev != dev or qn != n:
        raise L.MoeError("q: a row for each of x's, on its device")
    _scales(sq, "sq", n, K, dev)
    _call(L.lib().ainfer_moe_act_quant_fp8, dev, stream, x.data_ptr(), ld, dt, _live(live, dev), n,
          K, _kind(pow2), q.data_ptr(), qld, sq.data_ptr())
    return q, sq


def silu_mul_fp8(gate, up, q=None, sq=None, pow2=False, live=None, stream=None):
    """e4m3 codes and scales of gate / (1 + exp(-gate)) * up (ainfer_moe_silu_mul_fp8), as
    act_quant_fp8 writes them."""
    dt, dev, n, I, gld = _rows(gate, "gate")
    udt, udev, un, _, uld = _rows(up, "up", I)
    if not (udt == dt and un == n and udev == dev):
        raise L.MoeError("gate and up: one shape, type and device")
    if (q is None) != (sq is None):
        raise L.MoeError("q and sq: both or neither")
    if q is None:
        with _on(stream):
            q, sq = _new_codes(n, I, gate.device)
    qdev, qn, _, qld = _codes(q, "q", I)
    if qdev != dev or qn != n:
        raise L.MoeError("q: a row for each of gate's, on its device")
    _scales(sq, "sq", n, I, dev)
    _call(L.lib().ainfer_moe_silu_mul_fp8, dev, stream, gate.data_ptr(), gld, up.data_ptr(), uld, dt,
          _live(live, dev), n, I, _kind(pow2), q.data_ptr(), qld, sq.data_ptr())
    return q, sq


def silu_mul_backward(dact, gate, up, dgate, dup, live=None, stream=None):
    """The gradients of silu_mul to gate and up (ainfer_moe_silu_mul_backward), rows of
    any pitch and one type; dgate and dup may be dact, gate or up."""
    dt, dev, n, I, dld = _rows(dact, "dact")
    args = [dact.data_ptr(), dld]
    for t, name in ((gate, "gate"), (up, "up"), (dgate, "dgate"), (dup, "dup")):
        tdt, tdev, tn, _, ld = _rows(t, name, I)
        if not (tdt == dt and tdev == dev and tn == n):
            raise L.MoeError("dact, gate, up, dgate and dup: one shape, type and device")
        args += [t.data_ptr(), ld]
    _call(L.lib().ainfer_moe_silu_mul_backward, dev, stream, *args[:6], dt, _live(live, dev), n, I,
          *args[6:])
    return dgate, dup


def weight_quant_fp8(w, pow2=False, stream=None):
    """e4m3 codes [E][M][K] and scales [E][ceil(M / 128)][ceil(K / 128)] of w [E][M][K] fp32 or
    bf16 (ainfer_moe_weight_quant_fp8)."""
    dev = w.get_device()
    if not (w.dtype in _ACT and w.dim() == 3 and dev >= 0 and w.is_contiguous()):
        raise L.MoeError("w: contiguous [E][M][K] fp32 or bf16 on a device")
    E, M, K = w.shape
    with _on(stream):
        q = torch.empty(E, M, K, dtype=torch.float8_e4m3fn, device=w.device)
        s = torch.empty(E, -(-M // 128), -(-K // 128), dtype=torch.float32, device=w.device)
    _call(L.lib().ainfer_moe_weight_quant_fp8, dev, stream, w.data_ptr(), _ACT[w.dtype], E, M, K,
          _kind(pow2), q.data_ptr(), s.data_ptr())
    return q, s


class Fp8Weights:
    """The weights of E experts' projection (or one matrix, E = 1), resident on one
    device: e4m3 codes w [E][M][K] (float8_e4m3fn or uint8) laid out for the product
    (w itself is not kept), and their fp32 scales [E][ceil(M / 128)][ceil(K / 128)] (kept).
    transpose: the weights are W^T, [E][K][M], for the gradient to x (M a multiple of 16).
    stream: where they are laid out, behind what is on it; w may be dropped at once, products
    on other streams have to wait for it."""

    def __init__(self, w, scales, y_dtype=torch.bfloat16, transpose=False, stream=None):
        dev = w.get_device()
        if not (w.dtype in _CODES and w.dim() == 3 and dev >= 0 and w.is_contiguous()):
            raise L.MoeError("w: contiguous [E][M][K] codes on a device")
        E, M, K = w.shape
        if not (scales.dtype == torch.float32 and scales.get_device() == dev
                and scales.shape == (E, -(-M // 128), -(-K // 128)) and scales.is_contiguous()):
            raise L.MoeError("scales: contiguous fp32 [E][ceil(M / 128)][ceil(K / 128)] beside w")
        if y_dtype not in _ACT:
            raise L.MoeError("y: fp32 or bf16")
        if transpose:
            M, K = K, M
        n = L.lib().ainfer_moe_fp8_packed_bytes(E, M, K)
        if n == 0:
            raise L.MoeError("weight sizes outside the supported range")
        with torch.cuda.device(dev), _on(stream):
            self.packed = torch.empty(n, dtype=torch.uint8, device=w.device)
            self.scales = scales.transpose(1, 2).contiguous() if transpose else scales
        _call(L.lib().ainfer_moe_fp8_pack, dev, stream, w.data_ptr(), E, M, K, int(transpose),
              self.packed.data_ptr(), n)
        if stream is not None:  # their memory is not given out again before it has been read
            w.record_stream(stream)
            scales.record_stream(stream)
        self.shape, self.dev, self.y_dtype = (E, M, K), dev, y_dtype
        self.structs = {dt: L.Fp8(E, M, K, code, self.packed.data_ptr(), self.scales.data_ptr())
                        for dt, code in _ACT.items()}

    def product(self, q, sq, y=None, offsets=None, stream=None):
        """y [N][M] = x W^T for codes q [N][K] and scales sq of rows sorted by expert
        (offsets [E + 1] int32; may be left out with one expert), in fp32 or bf16
        (ainfer_moe_fp8_product).  Rows outside the offsets keep what y holds (a new y has
        anything there)."""
        E, M, K = self.shape
        dev, n, _, ld = _codes(q, "q", K)
        if dev != self.dev:
            raise L.MoeError("q: on the weights' device")
        _scales(sq, "sq", n, K, dev)
        if offsets is None:
            if E != 1:
                raise L.MoeError("offsets: the experts' rows")
        else:
            _vector(offsets, "offsets", torch.int32, E + 1, dev)
        if y is None:
            with _on(stream):
                y = torch.empty(n, M, dtype=self.y_dtype, device=q.device)
        _, ydev, yn, _, yld = _rows(y, "y", M)
        if ydev != dev or yn != n:
            raise L.MoeError("y: a row for each of q's, on its device")
        _call(L.lib().ainfer_moe_fp8_product, dev, stream, C.byref(self.structs[y.dtype]),
              q.data_ptr(), ld, sq.data_ptr(), offsets.data_ptr() if offsets is not None else None,
              n, y.data_ptr(), yld)
        return y


# ---- tokens sorted by expert and back --------------------------------------------
def sort_workspace(max_tokens, top_k, n_experts, device="cuda"):
    """Scratch of sort_rows with up to max_tokens tokens (no initialisation)."""
    n = L.lib().ainfer_moe_sort_workspace_bytes(max_tokens, top_k, n_experts)
    if n == 0:
        raise L.MoeError("invalid sizes for a sort workspace")
    ws = torch.empty(n + 256, dtype=torch.uint8, device=device)
    off = (-ws.data_ptr()) % 256
    return ws[off:off + n]


@functools.lru_cache(maxsize=256)
def _sorting(*fields):
    """The description of sorts of these sizes and types."""
    return L.Sorting(*fields)


def sort_rows(x, idx, n_experts, ws, fp8=False, pow2=False, out=None, stream=None):
    """The rows of x [T][H] in the order of their experts (idx [T][k] int32; ids outside
    [0, n_experts) are dropped): (rows [T * k][H], row_scales or None, offsets [E + 1], pos
    [T][k]) (ainfer_moe_sort_rows).  fp8: rows as e4m3 codes with their scales.  out: the
    four tensors to write; its rows' type then decides instead of fp8."""
    dt, dev, T, H, ld = _rows(x, "x")
    if not (idx.dtype == torch.int32 and idx.dim() == 2 and idx.shape[0] == T
            and idx.get_device() == dev and idx.is_contiguous()):
        raise L.MoeError("idx: contiguous int32 [T][k] on x's device")
    if ws.get_device() != dev or not ws.is_contiguous():
        raise L.MoeError("ws: on x's device")
    k = idx.shape[1]
    if out is None:
        with _on(stream):
            if fp8:
                rows, sc = _new_codes(T * k, H, x.device)
            else:
                rows, sc = torch.empty(T * k, H, dtype=x.dtype, device=x.device), None
            offsets = torch.empty(n_experts + 1, dtype=torch.int32, device=x.device)
            pos = torch.empty(T, k, dtype=torch.int32, device=x.device)
    else:
        rows, sc, offsets, pos = out
        fp8 = rows.dtype in _CODES
    if fp8:
        rdev, rn, _, rld = _codes(rows, "rows", H)
        if sc is None:
            raise L.MoeError("row_scales: fp32, beside rows of codes")
        _scales(sc, "row_scales", T * k, H, dev)
    else:
        _, rdev, rn, _, rld = _rows(rows, "rows", H)
        if rows.dtype != x.dtype or sc is not None:
            raise L.MoeError("rows: x's type without scales, or codes with them")
    if rdev != dev or rn != T * k:
        raise L.MoeError("rows: T * k of them, on x's device")
    _vector(offsets, "offsets", torch.int32, n_experts + 1, dev)
    if not (pos.dtype == torch.int32 and pos.shape == (T, k) and pos.get_device() == dev
            and pos.is_contiguous()):
        raise L.MoeError("pos: contiguous int32 [T][k] on x's device")
    d = _sorting(n_experts, k, H, dt, int(fp8), _kind(pow2))
    _call(L.lib().ainfer_moe_sort_rows, dev, stream, C.byref(d), x.data_ptr(), ld, idx.data_ptr(), T,
          offsets.data_ptr(), pos.data_ptr(), rows.data_ptr(), rld,
          sc.data_ptr() if fp8 else None, ws.data_ptr(), ws.nbytes)
    return rows, sc, offsets, pos


def _pairs(pos, w, T, dev):
    """k of pos [T][k] (and w [T][k], or None) on device dev."""
    if not (pos.dtype == torch.int32 and pos.dim() == 2 and pos.shape[0] == T
            and pos.get_device() == dev and pos.is_contiguous()):
        raise L.MoeError("pos: contiguous int32 [T][k] on the rows' device")
    if w is not None and not (w.dtype == torch.float32 and w.shape == pos.shape
                              and w.get_device() == dev and w.is_contiguous()):
        raise L.MoeError("w: contiguous fp32, of pos's shape, on its device")
    return pos.shape[1]


def unpermute(rows, pos, w, y, resid=None, stream=None):
    """y[t] = sum_j w[t][j] rows[pos[t][j]] (+ resid[t]) (ainfer_moe_unpermute); w None: 1,
    the gradient of sort_rows to x.  resid may be y."""
    rdt, dev, n, H, rld = _rows(rows, "rows")
    ydt, ydev, T, _, yld = _rows(y, "y", H)
    k = _pairs(pos, w, T, dev)
    if ydev != dev:
        raise L.MoeError("y: on the rows' device")
    sld = 0
    if resid is not None:
        sdt, sdev, sT, _, sld = _rows(resid, "resid", H)
        if not (sdt == ydt and sdev == dev and sT == T):
            raise L.MoeError("resid: y's shape, type and device")
    _call(L.lib().ainfer_moe_unpermute, dev, stream, rows.data_ptr(), rld, rdt, n, pos.data_ptr(),
          w.data_ptr() if w is not None else None, T, k, H,
          resid.data_ptr() if resid is not None else None, sld, y.data_ptr(), yld, ydt)
    return y


def unpermute_backward(dy, rows, pos, w, drows=None, dw=None, stream=None):
    """drows[pos[t][j]] = w[t][j] dy[t] and dw[t][j] = <dy[t], rows[pos[t][j]]>
    (ainfer_moe_unpermute_backward), in drows and dw; one that is None is left out."""
    ydt, dev, T, H, yld = _rows(dy, "dy")
    rdt, rdev, n, _, rld = _rows(rows, "rows", H)
    k = _pairs(pos, w, T, dev)
    if rdev != dev:
        raise L.MoeError("rows: on dy's device")
    dld = 0
    if drows is not None:
        ddt, ddev, dn, _, dld = _rows(drows, "drows", H)
        if not (ddt == rdt and ddev == dev and dn == n):
            raise L.MoeError("drows: the rows' shape, type and device")
    if dw is not None and not (dw.dtype == torch.float32 and dw.shape == pos.shape
                               and dw.get_device() == dev and dw.is_contiguous()):
        raise L.MoeError("dw: contiguous fp32, of pos's shape, on its device")
    _call(L.lib().ainfer_moe_unpermute_backward, dev, stream, dy.data_ptr(), yld, ydt,
          rows.data_ptr(), rld, rdt, n, pos.data_ptr(), w.data_ptr() if w is not None else None, T,
          k, H, drows.data_ptr() if drows is not None else None, dld,
          dw.data_ptr() if dw is not None else None)
    return drows, dw


class Fp8Experts:
    """The routed experts' MLP with 8-bit floating point weights: gate_up [E][2 I][H]
    (gate rows, then up rows) and down [E][H][I], Fp8Weights on one device.  Takes the
    routing of route_scored or MoeLayer.route; ids outside [0, E) (experts of other GPUs)
    add nothing.  back: the two transposed, Fp8Weights(..., transpose=True), for backward."""

    def __init__(self, gate_up, down, back=None, pow2=False):
        E, I2, H = gate_up.shape
        I = I2 // 2
        if down.shape != (E, H, I) or I2 % 2 or gate_up.dev != down.dev:
            raise L.MoeError("gate_up [E][2 I][H] and down [E][H][I] on one device")
        if back is not None and not (back[0].shape == (E, H, I2) and back[1].shape == (E, I, H)
                                     and back[0].dev == back[1].dev == down.dev):
            raise L.MoeError("back: gate_up and down transposed, beside them")
        self.gate_up, self.down, self.back, self.pow2 = gate_up, down, back, pow2
        self.n_experts, self.inter, self.hidden = E, I, H

    def _check(self, x, idx, w, y, resid):
        """(T, k); every tensor of a call, before the first kernel is enqueued."""
        _, dev, T, _, _ = _rows(x, "x", self.hidden)
        if dev != self.gate_up.dev:
            raise L.MoeError("x: on the experts' device")
        for t, name, dt in ((idx, "idx", torch.int32), (w, "w", torch.float32)):
            if not (t.dtype == dt and t.dim() == 2 and t.shape[0] == T and t.shape == idx.shape
                    and t.get_device() == dev and t.is_contiguous()):
                raise L.MoeError(f"{name}: contiguous {dt} [T][k] on x's device")
        for t, name in ((y, "y"), (resid, "resid")):
            if t is not None:
                _, tdev, n, _, _ = _rows(t, name, self.hidden)
                if tdev != dev or n != T:
                    raise L.MoeError(f"{name}: a row for each of x's, on its device")
        if resid is not None and resid.dtype != (x if y is None else y).dtype:
            raise L.MoeError("resid: y's type")
        return idx.shape

    def forward(self, x, idx, w, y=None, resid=None, stream=None, keep=False):
        """y[t] = sum_j w[t][j] expert_{idx[t][j]}(x[t]) (+ resid[t]), x and y [T][H] bf16 or
        fp32 rows: rows sorted and quantised, gate and up, gated activation quantised,
        down, weighted sums.  y and resid may be x.  keep: (y, what backward needs) instead of
        y; backward is to run on the same stream, or behind it."""
        T, k = self._check(x, idx, w, y, resid)
        I, dev = self.inter, self.gate_up.dev
        with torch.cuda.device(dev), _on(stream):
            ws = sort_workspace(T, k, self.n_experts, x.device)
            q, sq, offsets, pos = sort_rows(x, idx, self.n_experts, ws, fp8=True, pow2=self.pow2)
            h = self.gate_up.product(q, sq, offsets=offsets)
            a, sa = silu_mul_fp8(h[:, :I], h[:, I:], pow2=self.pow2, live=offsets)
            o = self.down.product(a, sa, offsets=offsets)
            if y is None:
                y = torch.empty_like(x)
            unpermute(o, pos, w, y, resid)
        return (y, (h, o, offsets, pos, w)) if keep else y

    def backward(self, dy, kept, stream=None, resid=None):
        """(dx [T][H] of dy's type, dw [T][k] fp32) from dy [T][H] and forward's kept
        tensors.  dx is the experts' share alone: the gradient of forward's resid is dy.  resid
        [T][H] of dy's type is added to dx before it is rounded: dy itself where forward's
        resid was x.  The weights are constants; the products' gradients are quantised to
        e4m3 as the activations are, and each rounding passes its gradient on."""
        if self.back is None:
            raise L.MoeError("experts with transposed weights (back)")
        h, o, offsets, pos, w = kept
        if resid is not None:
            _, rdev, n, _, _ = _rows(resid, "resid", self.hidden)
            if not (resid.dtype == dy.dtype and rdev == dy.get_device() and n == dy.shape[0]):
                raise L.MoeError("resid: dy's shape, type and device")
        I = self.inter
        with torch.cuda.device(self.gate_up.dev), _on(stream):
            do, dw = unpermute_backward(dy, o, pos, w, torch.empty_like(o), torch.empty_like(w))
            q, sq = act_quant_fp8(do, pow2=self.pow2, live=offsets)
            dact = self.back[1].product(q, sq, offsets=offsets,
                                        y=torch.empty(len(q), I, dtype=h.dtype, device=h.device))
            dh = torch.empty_like(h)
            silu_mul_backward(dact, h[:, :I], h[:, I:], dh[:, :I], dh[:, I:], live=offsets)
            q, sq = act_quant_fp8(dh, pow2=self.pow2, live=offsets)
            drows = self.back[0].product(q, sq, offsets=offsets)
            dx = unpermute(drows, pos, None, torch.empty_like(dy), resid)
        return dx, dw
