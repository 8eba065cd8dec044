"""Tensor-level wrappers of the evamx C ABI (PyTorch-ROCm tensors in, device pointers out).

Every function launches HIP kernels from libevamx.so on the current stream; nothing here
computes on the CPU.
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import MoeArgs, MoeShape, W4Desc, W4MoeArgs, check, lib, ptr, stream_handle

SCORE_FNS = {"sigmoid": _lib.SCORE_SIGMOID, "sqrt_softplus": _lib.SCORE_SQRT_SOFTPLUS}
RATES = (2.0, 3.0, 4.0, 5.0)


def _dev(t: torch.Tensor, name: str, dtype=None, ndim=None, row_strided=False):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if ndim is not None and t.ndim != ndim:
        raise ValueError(f"{name} must have {ndim} dims")
    if row_strided:
        if t.stride(-1) != 1 or (t.ndim == 2 and t.stride(0) < t.shape[1]):
            raise ValueError(f"{name} must have unit column stride and non-overlapping rows")
    elif not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def tile_u16(bits: float) -> int:
    b = float(bits)
    return 16 * int(b) + 8 if b != int(b) else 16 * int(b)


def exl3_dequant(trellis: torch.Tensor, bits: float) -> torch.Tensor:
    """fp16 ``W[in][out]`` of an EXL3 projection ``trellis int16 [in/16, out/16, T]``."""
    _dev(trellis, "trellis", torch.int16, 3)
    kt, nt, t16 = trellis.shape
    if t16 != tile_u16(bits):
        raise ValueError(f"trellis last dim {t16} does not match {bits} bits")
    w = torch.empty(kt * 16, nt * 16, dtype=torch.float16, device=trellis.device)
    check(lib().evamx_exl3_dequant(ptr(trellis), kt * 16, nt * 16, float(bits), ptr(w),
                                   stream_handle(trellis.device)), "evamx_exl3_dequant")
    return w


def exl3_linear(x: torch.Tensor, trellis: torch.Tensor, suh: torch.Tensor, svh: torch.Tensor, bits: float,
                out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Single EXL3 linear, fp16 ``x [M, in]`` -> fp16 ``[M, out]`` (decode GEMV up to 16 rows, MFMA
    tiles beyond)."""
    _dev(x, "x", torch.float16, 2)
    _dev(trellis, "trellis", torch.int16, 3)
    _dev(suh, "suh", torch.float16, 1)
    _dev(svh, "svh", torch.float16, 1)
    m, n_in = x.shape
    n_out = svh.numel()
    if suh.numel() != n_in or trellis.shape[0] * 16 != n_in or trellis.shape[1] * 16 != n_out:
        raise ValueError("x / trellis / suh / svh shapes disagree")
    if out is None:
        out = torch.empty(m, n_out, dtype=torch.float16, device=x.device)
    _dev(out, "out", torch.float16, 2)
    if tuple(out.shape) != (m, n_out):
        raise ValueError(f"out must be [{m}, {n_out}]")
    need = lib().evamx_exl3_linear_workspace_bytes(m, n_in, n_out)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    _dev(workspace, "workspace", torch.uint8, 1)
    check(lib().evamx_exl3_linear(ptr(x), m, n_in, n_out, ptr(trellis), ptr(suh), ptr(svh), float(bits), ptr(out),
                                  ptr(workspace), workspace.numel(), stream_handle(x.device)), "evamx_exl3_linear")
    return out


class W4Weight:
    """A stack of 4-bit matrices with group scales in the layout the kernels read (``w4_pack`` makes it):
    ``W[n, k] = scale[n, k // group] * (code[n, k] - zero[n, k // group])``, zero 8 without zero points."""

    def __init__(self, count: int, n_out: int, n_in: int, group: int, scale_dtype: torch.dtype, zeros: bool, device):
        stored = lib().evamx_w4_stored_group(group)
        if stored == 0:
            raise ValueError(f"group {group} is not a positive multiple of 32")
        if scale_dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("scales must be fp16 or bf16")
        nbytes, groups = lib().evamx_w4_code_bytes(count, n_out, n_in), lib().evamx_w4_group_count(count, n_out, n_in, stored)
        if nbytes == 0:
            raise ValueError(f"{count} matrices [{n_out}, {n_in}] outside 1..{_lib.W4_MAX_COUNT} and 1..{_lib.W4_MAX_DIM}")
        self.count, self.n_out, self.n_in, self.group = count, n_out, n_in, group
        self.codes = torch.empty(nbytes, dtype=torch.uint8, device=device)
        self.device = self.codes.device                      # with its index, whatever `device` names
        self.scales = torch.empty(groups, dtype=scale_dtype, device=device)
        self.zeros = torch.empty(groups, dtype=torch.uint8, device=device) if zeros else None
        self.desc = W4Desc(ptr(self.codes), ptr(self.scales), ptr(self.zeros), count, n_out, n_in, stored,
                           _DTYPES[scale_dtype])


_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


def w4_pack(codes: torch.Tensor, scales: torch.Tensor, *, n_in: int, group: int, zeros: torch.Tensor | None = None) -> W4Weight:
    """Lay 4-bit weights out for ``w4_linear`` / ``w4_moe_forward``. ``codes`` uint8 ``[(count,) n_out,
    ceil(n_in / 2)]``, two codes of a row to a byte, the even one in the lower half; ``scales`` fp16 or
    bf16 ``[(count,) n_out, ceil(n_in / group)]``; ``zeros`` uint8 like the scales, the values that stand
    for zero (0..31, so also the 16 of formats that hold them less one; without them 8), read back to be checked
    unless in a graph capture. ``group``: a multiple of 32 input features that share a scale."""
    _dev(codes, "codes", torch.uint8)
    if codes.ndim not in (2, 3):
        raise ValueError("codes must be [n_out, ceil(n_in / 2)] or a stack of such")
    _dev(scales, "scales", None, codes.ndim)
    if group < 32 or group % 32:
        raise ValueError(f"group {group} is not a positive multiple of 32")
    lead, n_out = tuple(codes.shape[:-2]), codes.shape[-2]
    groups = (*lead, n_out, -(-n_in // group))
    if codes.shape[-1] != (n_in + 1) // 2 or tuple(scales.shape) != groups:
        raise ValueError(f"codes {tuple(codes.shape)} / scales {tuple(scales.shape)} disagree with n_in {n_in}, group {group}")
    if zeros is not None:
        _dev(zeros, "zeros", torch.uint8, codes.ndim)
        if tuple(zeros.shape) != groups:
            raise ValueError(f"zeros must have the scales' shape {groups}, got {tuple(zeros.shape)}")
        if zeros.numel() and not torch.cuda.is_current_stream_capturing() and int(zeros.max()) > _lib.W4_MAX_ZERO:
            raise ValueError(f"zero points up to {int(zeros.max())}: a weight takes 0..{_lib.W4_MAX_ZERO}")
    for t, name in ((scales, "scales"), (zeros, "zeros")):
        if t is not None and t.device != codes.device:
            raise ValueError(f"{name} is on {t.device}, the codes on {codes.device}")
    w = W4Weight(lead[0] if lead else 1, n_out, n_in, group, scales.dtype, zeros is not None, codes.device)
    _launch(lib().evamx_w4_pack, "evamx_w4_pack", w.device, ptr(codes), ptr(scales), ptr(zeros), group, ctypes.byref(w.desc))
    return w


def w4_dequant(weight: W4Weight) -> torch.Tensor:
    """fp32 ``[count, n_out, n_in]`` of packed 4-bit weights."""
    out = torch.empty(weight.count, weight.n_out, weight.n_in, dtype=torch.float32, device=weight.device)
    _launch(lib().evamx_w4_dequant, "evamx_w4_dequant", weight.device, ctypes.byref(weight.desc), ptr(out))
    return out


def _launch(fn, what: str, device: torch.device, *args):
    """One library call on the current stream of ``device``, which is made current if it is not."""
    if device.index == torch.cuda.current_device():
        check(fn(*args, torch._C._cuda_getCurrentRawStream(device.index)), what)
    else:
        with torch.cuda.device(device):
            check(fn(*args, torch._C._cuda_getCurrentRawStream(device.index)), what)


def _row_stride(t: torch.Tensor, name: str, dtype=None) -> int:
    """Row stride of a 2-dim device tensor whose rows are contiguous and do not overlap (a single row: any)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.ndim != 2:
        raise ValueError(f"{name} must be a 2-dim device tensor")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    rows, cols = t.shape
    if (cols > 1 and t.stride(1) != 1) or (rows > 1 and t.stride(0) < cols):
        raise ValueError(f"{name} must have unit column stride and non-overlapping rows")
    return t.stride(0) if rows > 1 else cols


def _no_grad(name, *tensors):
    """Refuses tensors whose derivatives autograd would expect ``name`` to carry on, backward or forward."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} has no backward: call it under torch.no_grad() or with detached tensors")
    if forward_ad._current_level >= 0 and not torch.is_inference_mode_enabled():      # no_grad does not switch forward mode off
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{name} has no forward-mode derivative: call it with the primal of {forward_ad.__name__}.unpack_dual")


def w4_linear(x: torch.Tensor, weight: W4Weight, bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ W.T + bias`` on 4-bit weights with group scales: ``x`` fp16 or bf16 ``[1..65536, n_in]``
    (rows of any stride), ``bias`` and the result of x's dtype, summed in fp32 and rounded once. ``out``
    must not overlap ``x``."""
    x_stride = _row_stride(x, "x")
    if x.dtype not in _DTYPES:
        raise ValueError("x must be fp16 or bf16")
    rows = x.shape[0]
    if weight.count != 1 or x.shape[1] != weight.n_in:
        raise ValueError(f"x {tuple(x.shape)} does not fit {weight.count} matrices [{weight.n_out}, {weight.n_in}]")
    if not 1 <= rows <= 65536:
        raise ValueError(f"x has {rows} rows, a call takes 1..65536")
    device = x.device
    if bias is not None:
        _dev(bias, "bias", x.dtype, 1)
        if bias.numel() != weight.n_out or bias.device != device:
            raise ValueError(f"bias must be [{weight.n_out}] on {device}")
    if out is None:
        out = torch.empty(rows, weight.n_out, dtype=x.dtype, device=device)
        out_stride = weight.n_out
    else:
        out_stride = _row_stride(out, "out", x.dtype)
        if tuple(out.shape) != (rows, weight.n_out) or out.device != device:
            raise ValueError(f"out must be [{rows}, {weight.n_out}] on {device}")
    _no_grad("w4_linear", x, bias, out)
    if workspace is None:
        workspace = torch.empty(lib().evamx_w4_linear_workspace_bytes(rows, weight.n_in), dtype=torch.uint8, device=device)
    else:
        _dev(workspace, "workspace", torch.uint8, 1)
    if weight.device != device or workspace.device != device:
        raise ValueError(f"x is on {device}, the weight on {weight.device}, the workspace on {workspace.device}")
    _launch(lib().evamx_w4_linear, "evamx_w4_linear", device, ptr(x), _DTYPES[x.dtype], x_stride, rows, ctypes.byref(weight.desc),
            ptr(bias), ptr(out), out_stride, ptr(workspace), workspace.numel())
    return out


def route_topk(logits: torch.Tensor, topk: int, score_fn: str = "sigmoid", sel_bias: torch.Tensor | None = None,
               route_scale: float = 1.0):
    """(indices int64, weights fp32, rw fp16) of the top-k experts per row of ``logits [T, E]``."""
    _dev(logits, "logits", torch.float32, 2)
    t, e = logits.shape
    if sel_bias is not None:
        _dev(sel_bias, "sel_bias", torch.float32, 1)
    idx = torch.empty(t, topk, dtype=torch.int64, device=logits.device)
    w = torch.empty(t, topk, dtype=torch.float32, device=logits.device)
    rw = torch.empty(t, topk, dtype=torch.float16, device=logits.device)
    check(lib().evamx_route_topk(ptr(logits), ptr(sel_bias), t, e, topk, SCORE_FNS[score_fn], float(route_scale),
                                 ptr(idx), ptr(w), ptr(rw), stream_handle(logits.device)), "evamx_route_topk")
    return idx, w, rw


def router_logits(x: torch.Tensor, gate_w: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """fp32 ``x.float() @ gate_w.T`` on the device (``evamx_router_logits``), each row reduced in one
    fixed order whatever the batch (model.py:158-165)."""
    if x.dim() != 2 or x.dtype not in (torch.float16, torch.bfloat16) or not x.is_cuda or x.stride(1) != 1:
        raise ValueError("x must be a CUDA fp16/bf16 [rows, hidden] tensor with unit inner stride")
    _dev(gate_w, "gate_w", torch.float32, 2)
    rows, hidden = x.shape
    if gate_w.shape[1] != hidden:
        raise ValueError(f"gate_w must be [n_experts, {hidden}]")
    if out is None:
        out = torch.empty(rows, gate_w.shape[0], dtype=torch.float32, device=x.device)
    _dev(out, "out", torch.float32, 2)
    check(lib().evamx_router_logits(ptr(x), _lib.DTYPE_BF16 if x.dtype == torch.bfloat16 else _lib.DTYPE_F16, x.stride(0), rows,
                                    ptr(gate_w), gate_w.shape[0], hidden, ptr(out), stream_handle(x.device)),
          "evamx_router_logits")
    return out


def route(x: torch.Tensor, gate_w: torch.Tensor, gate_b: torch.Tensor | None, topk: int, route_scale: float = 1.0,
          score_fn: str = "sqrt_softplus", image_mask: torch.Tensor | None = None,
          gate_b_vl: torch.Tensor | None = None):
    """``Block.route(x, image_mask) -> (w, idx)`` (model.py:404-416) on the device: gate GEMV, scores,
    top-k of score + bias (``gate_b_vl`` for the rows of ``image_mask``), weights normalised and
    scaled. With a mask both biases are routed and the rows picked by ``torch.where`` (no host sync)."""
    z = router_logits(x, gate_w)
    idx, w, _ = route_topk(z, topk, score_fn, gate_b, route_scale)
    if image_mask is not None and gate_b_vl is not None:
        idx_vl, w_vl, _ = route_topk(z, topk, score_fn, gate_b_vl, route_scale)
        m = image_mask.reshape(-1, 1).to(device=z.device, dtype=torch.bool)
        idx = torch.where(m, idx_vl, idx)
        w = torch.where(m, w_vl, w)
    return w, idx


_LOGIT_DTYPES = {torch.float32: _lib.DTYPE_F32, **_DTYPES}


def _balance_args(logits, score_fn, seq_starts, token_mask):
    """Checked (stride, sequences, starts, mask bytes) of a balance call."""
    stride = _row_stride(logits, "logits")
    if logits.dtype not in _LOGIT_DTYPES:
        raise ValueError("logits must be fp32, bf16 or fp16")
    if score_fn not in SCORE_FNS:
        raise ValueError(f"score_fn {score_fn!r} not in {sorted(SCORE_FNS)}")
    n = 1
    if seq_starts is not None:
        _dev(seq_starts, "seq_starts", torch.int32, 1)
        n = seq_starts.numel() - 1
        if n < 1:
            raise ValueError("seq_starts must hold the start of each sequence and the last one's end")
    if token_mask is not None:
        _dev(token_mask, "token_mask", torch.bool, 1)
        if token_mask.numel() != logits.shape[0]:
            raise ValueError(f"token_mask must be [{logits.shape[0]}]")
    for t, name in ((seq_starts, "seq_starts"), (token_mask, "token_mask")):
        if t is not None and t.device != logits.device:
            raise ValueError(f"{name} is on {t.device}, logits on {logits.device}")
    return stride, n


def _balance_forward(logits, sel, score_fn, stride, n, seq_starts, token_mask):
    """(loss, counts, tokens) for checked arguments."""
    rows, experts = logits.shape
    dev = logits.device
    _dev(sel, "sel", torch.int64, 2)
    if sel.shape[0] != rows or sel.device != dev:
        raise ValueError(f"sel must be [{rows}, topk] on {dev}, got {tuple(sel.shape)} on {sel.device}")
    loss = torch.empty(n, dtype=torch.float32, device=dev)
    counts = torch.empty(n, experts, dtype=torch.int32, device=dev)
    tokens = torch.empty(n, dtype=torch.int32, device=dev)
    ws = torch.empty(lib().evamx_balance_workspace_bytes(rows, experts, n), dtype=torch.uint8, device=dev)
    _launch(lib().evamx_balance_loss, "evamx_balance_loss", dev, ptr(logits), _LOGIT_DTYPES[logits.dtype], stride, rows, experts, ptr(sel),
            sel.shape[1], SCORE_FNS[score_fn], ptr(seq_starts), n, ptr(token_mask), ptr(loss), ptr(counts), ptr(tokens), ptr(ws), ws.numel())
    return loss, counts, tokens


def _balance_backward(grad_loss, logits, counts, tokens, topk, score_fn, stride, n, seq_starts, token_mask):
    """The logits' gradient for checked arguments."""
    rows, experts = logits.shape
    grad = torch.empty(rows, experts, dtype=logits.dtype, device=logits.device)
    _launch(lib().evamx_balance_grad, "evamx_balance_grad", logits.device, ptr(grad_loss), ptr(logits), _LOGIT_DTYPES[logits.dtype],
            stride, rows, experts, topk, SCORE_FNS[score_fn], ptr(seq_starts), n, ptr(token_mask), ptr(counts), ptr(tokens), ptr(grad))
    return grad


def balance_stats(logits: torch.Tensor, sel: torch.Tensor, *, score_fn: str = "sigmoid", seq_starts: torch.Tensor | None = None,
                  token_mask: torch.Tensor | None = None):
    """``(loss fp32 [S], counts int32 [S, E], tokens int32 [S])`` of ``balance_loss``, outside autograd."""
    stride, n = _balance_args(logits, score_fn, seq_starts, token_mask)
    return _balance_forward(logits, sel, score_fn, stride, n, seq_starts, token_mask)


def balance_loss_grad(grad_loss: torch.Tensor, logits: torch.Tensor, counts: torch.Tensor, tokens: torch.Tensor, topk: int, *,
                      score_fn: str = "sigmoid", seq_starts: torch.Tensor | None = None,
                      token_mask: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of ``(grad_loss * loss).sum()`` with respect to the logits, for the ``counts`` and
    ``tokens`` that ``balance_stats`` gave for the same arguments; zero for rows that do not count."""
    stride, n = _balance_args(logits, score_fn, seq_starts, token_mask)
    for t, name, dtype, shape in ((grad_loss, "grad_loss", torch.float32, (n,)), (counts, "counts", torch.int32, (n, logits.shape[1])),
                                  (tokens, "tokens", torch.int32, (n,))):
        _dev(t, name, dtype)
        if tuple(t.shape) != shape or t.device != logits.device:
            raise ValueError(f"{name} must be {shape} on {logits.device}, got {tuple(t.shape)} on {t.device}")
    return _balance_backward(grad_loss, logits, counts, tokens, topk, score_fn, stride, n, seq_starts, token_mask)


_NO_CAPTURE = "balance_loss is not captured with a backward pass: call balance_stats and balance_loss_grad"


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, sel, score_fn, seq_starts, token_mask):
        stride, n = _balance_args(logits, score_fn, seq_starts, token_mask)
        loss, counts, tokens = _balance_forward(logits, sel, score_fn, stride, n, seq_starts, token_mask)
        ctx.save_for_backward(logits, counts, tokens, seq_starts, token_mask)
        ctx.args = sel.shape[1], score_fn, stride, n
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)                 # no zeros for the counts, which have no gradient
        return loss, counts

    @staticmethod
    def backward(ctx, grad_loss, _):
        if grad_loss is None:
            return None, None, None, None, None
        if torch.is_grad_enabled():                      # create_graph=True: a gradient without a graph would pass for a constant
            raise RuntimeError("balance_loss is differentiable once")
        if torch.cuda.is_current_stream_capturing():     # of a forward pass that was not
            raise RuntimeError(_NO_CAPTURE)
        logits, counts, tokens, seq_starts, token_mask = ctx.saved_tensors
        return _balance_backward(grad_loss.contiguous(), logits, counts, tokens, *ctx.args, seq_starts, token_mask), None, None, None, None


def balance_loss(logits: torch.Tensor, sel: torch.Tensor, *, score_fn: str = "sigmoid", seq_starts: torch.Tensor | None = None,
                 token_mask: torch.Tensor | None = None):
    """Balance loss of each sequence and the picks of each expert, ``(loss fp32 [S], counts int32 [S, E])``,
    for router ``logits [T, E]`` (fp32, bf16 or fp16) and their routes ``sel`` int64 ``[T, topk]`` (``route_topk``).

    With ``p = score / score.sum(1)``, ``n`` tokens and ``c_e`` picks of expert e in a sequence, the loss is
    ``sum_e (E c_e / (topk n)) (sum_t p_te / n)``: 1 where picks and shares are even, larger where the experts
    that are picked often also have large scores. It is differentiable in the logits, for a program whose own
    product makes them (``router_logits`` and ``route`` have no backward pass: behind them ``balance_stats`` gives
    the same numbers); the counts (which serve a selection bias as well as the loss) are constants. ``seq_starts`` int32 ``[S + 1]`` ascending: sequence
    s is rows ``seq_starts[s]`` to ``seq_starts[s + 1]``, and rows of none count nowhere; without it all rows
    are one sequence. ``token_mask`` bool ``[T]``: rows that count. A sequence without such rows has loss 0.
    Picks outside ``[0, E)`` are not counted.

    The backward pass is not for a graph capture (autograd's own streams and accumulators are not): there call
    ``balance_stats`` and ``balance_loss_grad``. It is refused there and with ``create_graph=True``: there is no
    second derivative."""
    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad and logits.is_cuda and \
            torch.cuda.is_current_stream_capturing():
        raise RuntimeError(_NO_CAPTURE)
    return _BalanceLoss.apply(logits, sel, score_fn, seq_starts, token_mask)


def prepare_routes_workspace_bytes(capacity: int, topk: int) -> int:
    n = lib().evamx_prepare_routes_workspace_bytes(capacity, topk)
    if n == 0:
        raise ValueError("invalid capacity/topk")
    return n


def prepare_routes(sel: torch.Tensor, rw: torch.Tensor, capacity: int, n_local: int,
                   runs: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """The reference run table ``int32 [2 + 2*capacity*topk + 1]`` for routes ``sel``/``rw`` (fp16)."""
    _dev(sel, "sel", torch.int64, 2)
    _dev(rw, "rw", torch.float16, 2)
    t, k = sel.shape
    if rw.shape != sel.shape:
        raise ValueError("sel/rw shapes differ")
    if runs is None:
        runs = torch.empty(2 + 2 * capacity * k + 1, dtype=torch.int32, device=sel.device)
    need = lib().evamx_prepare_routes_workspace_bytes(capacity, k)
    if workspace is None:
        workspace = torch.zeros(need, dtype=torch.uint8, device=sel.device)
    check(lib().evamx_prepare_routes(ptr(sel), ptr(rw), t, k, capacity, n_local, ptr(runs), ptr(workspace),
                                     workspace.numel(), stream_handle(sel.device)), "evamx_prepare_routes")
    return runs


class MoeWorkspace:
    """Device workspace of the MoE forward for one shape (owned by one runner)."""

    def __init__(self, device, rows_max: int, hidden: int, inter: int, topk: int, n_local: int,
                 has_shared: bool, ksplit_gu: int = 0, ksplit_down: int = 0, strict_rows: int = 0):
        """``strict_rows`` > 0: calls of up to that many rows give every row the bits it gets in a
        one-row call (strict batch mode, the reference's DS41_STRICT_BATCH); 0: automatic geometry."""
        self.shape = MoeShape(rows_max, hidden, inter, topk, n_local, int(bool(has_shared)), ksplit_gu, ksplit_down,
                              strict_rows)
        nbytes = lib().evamx_moe_workspace_bytes(ctypes.byref(self.shape))
        if nbytes == 0:
            raise ValueError("invalid MoE shape: " + lib().evamx_last_error().decode())
        self.device = torch.device(device)
        self.buffer = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        check(lib().evamx_moe_workspace_init(ctypes.byref(self.shape), ptr(self.buffer), stream_handle(self.device)),
              "evamx_moe_workspace_init")

    def clear_flags(self) -> None:
        """Zero the sticky device flag word (a fill kernel on the current stream)."""
        check(lib().evamx_moe_workspace_init(ctypes.byref(self.shape), ptr(self.buffer), stream_handle(self.device)),
              "evamx_moe_workspace_init")

    def runs(self) -> torch.Tensor:
        """View of the run table written by the last forward."""
        slots = self.shape.rows_max * self.shape.topk
        addr = lib().evamx_moe_runs_ptr(ctypes.byref(self.shape), ptr(self.buffer))
        off = addr - self.buffer.data_ptr()
        n = 2 + 2 * slots + 1
        return self.buffer[off:off + 4 * n].view(torch.int32)

    def logits(self, rows: int, n_logits: int) -> torch.Tensor:
        """fp32 ``[rows, n_logits]`` router logits the last forward computed from ``gate_w``."""
        addr = lib().evamx_moe_logits_ptr(ctypes.byref(self.shape), ptr(self.buffer))
        off = addr - self.buffer.data_ptr()
        return self.buffer[off:off + 4 * rows * n_logits].view(torch.float32).view(rows, n_logits)

    def rotated(self) -> torch.Tensor:
        """fp16 ``[2, nslot_max, hidden]`` view of the rotated gate (0) and up (1) inputs the last
        forward of 3 or more rows wrote: routed slot ``row * topk + k``, shared-expert row ``r`` at
        ``rows * topk + r``."""
        s = self.shape
        nslot_max = s.rows_max * s.topk + (s.rows_max if s.has_shared else 0)
        addr = lib().evamx_moe_rotated_ptr(ctypes.byref(s), ptr(self.buffer))
        off = addr - self.buffer.data_ptr()
        n = 2 * nslot_max * s.hidden
        return self.buffer[off:off + 2 * n].view(torch.float16).view(2, nslot_max, s.hidden)

    def flags(self) -> torch.Tensor:
        addr = lib().evamx_moe_flags_ptr(ctypes.byref(self.shape), ptr(self.buffer))
        off = addr - self.buffer.data_ptr()
        return self.buffer[off:off + 4].view(torch.int32)


def _check_forward_args(s, device, x, tables, out, bits, k2_per_expert, logits, sel, weights, rw, sel_bias,
                        shared_ptrs, shared_bits, events, residual, gate_w):
    """Every tensor's device, dtype and shape against the workspace's shape, before any launch:
    the C ABI receives bare pointers and would read or write out of bounds otherwise."""
    def on_dev(t, name, dtype, shape=None, row_strided=False):
        _dev(t, name, dtype, len(shape) if shape is not None else None, row_strided=row_strided)
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, the workspace on {device}")
        if shape is not None:
            for i, (have, want) in enumerate(zip(t.shape, shape)):
                if want is not None and have != want:
                    raise ValueError(f"{name} must have shape {tuple('*' if w is None else w for w in shape)}, "
                                     f"got {tuple(t.shape)}")

    on_dev(x, "x", None, (None, s.hidden), row_strided=True)
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("x must be fp16 or bf16")
    rows, topk = x.shape[0], s.topk
    if not 1 <= rows <= s.rows_max:
        raise ValueError(f"x has {rows} rows, the workspace holds 1..{s.rows_max}")
    on_dev(tables, "tables", torch.int64, (9, s.n_local))
    if out is None and residual is None:
        raise ValueError("need out, residual or both")
    if out is not None:
        on_dev(out, "out", torch.float32, (None, None), row_strided=True)
        if out.shape[0] < rows or out.shape[1] < s.hidden:
            raise ValueError(f"out must be at least [{rows}, {s.hidden}], got {tuple(out.shape)}")
    if residual is not None:
        on_dev(residual, "residual", torch.bfloat16, (rows, None), row_strided=True)
        if residual.shape[1] < s.hidden:
            raise ValueError(f"residual must be [{rows}, >= {s.hidden}]")
    if sel is None:
        raise ValueError("sel is required (routes in, or the routing's output)")
    on_dev(sel, "sel", torch.int64, (rows, topk))
    if weights is not None:
        on_dev(weights, "weights", torch.float32, (rows, topk))
    if rw is not None:
        on_dev(rw, "rw", torch.float16, (rows, topk))
    if logits is not None and gate_w is not None:
        raise ValueError("give logits or gate_w, not both")
    routing = logits is not None or gate_w is not None
    if routing:
        if weights is None:
            raise ValueError("routing on the device writes weights: pass an fp32 [rows, topk] output")
        if logits is not None:
            on_dev(logits, "logits", torch.float32, (rows, None))
            n_logits = logits.shape[1]
        else:
            on_dev(gate_w, "gate_w", torch.float32, (None, s.hidden))
            n_logits = gate_w.shape[0]
        if not topk <= n_logits <= 512:
            raise ValueError(f"{n_logits} experts in the router, need {topk}..512")
        if sel_bias is not None:
            on_dev(sel_bias, "sel_bias", torch.float32, (n_logits,))
    elif weights is None and rw is None:
        raise ValueError("given routes need fp32 weights or fp16 rw")
    elif sel_bias is not None:
        raise ValueError("sel_bias applies only when routing on the device")
    if k2_per_expert is not None:
        on_dev(k2_per_expert, "k2_per_expert", torch.uint8, (s.n_local,))
    elif bits is None:
        raise ValueError("give a uniform rate (bits) or k2_per_expert")
    if s.has_shared:
        if shared_ptrs is None or len(shared_ptrs) != 9 or shared_bits is None:
            raise ValueError("the workspace has a shared expert: pass its 9 pointers and shared_bits")
    elif shared_ptrs is not None:
        raise ValueError("the workspace was built without a shared expert")
    if events is not None and len(events) != 10:
        raise ValueError("events must hold 10 event handles")


def _moe_args(s, device, x, tables, out, limit, bits, k2_per_expert, logits, sel, weights, rw, score_fn, sel_bias,
              route_scale, shared_ptrs, shared_bits, min_expert, max_expert, events, residual, gate_w,
              bits_down=None, k2_down_per_expert=None, shared_bits_down=None, shared_gate_w=None):
    """The evamx_moe_args of one forward call (every tensor checked first), without the
    workspace; returns it with the ctypes array of shared pointers it refers to."""
    _check_forward_args(s, device, x, tables, out, bits, k2_per_expert, logits, sel, weights, rw, sel_bias,
                        shared_ptrs, shared_bits, events, residual, gate_w)
    if k2_down_per_expert is not None:
        _dev(k2_down_per_expert, "k2_down_per_expert", torch.uint8, 1)
        if k2_down_per_expert.device != device or k2_down_per_expert.numel() != s.n_local:
            raise ValueError(f"k2_down_per_expert must be a uint8 [{s.n_local}] tensor on {device}")
    if shared_gate_w is not None:
        _dev(shared_gate_w, "shared_gate_w", torch.float16, 1)
        if shared_gate_w.device != device or shared_gate_w.numel() != s.hidden:
            raise ValueError(f"shared_gate_w must be an fp16 [{s.hidden}] tensor on {device}")
        if not s.has_shared:
            raise ValueError("shared_gate_w needs a shared expert")
    a = MoeArgs()
    a.shape = s
    a.rows = x.shape[0]
    a.x = ptr(x)
    a.x_dtype = _lib.DTYPE_F16 if x.dtype == torch.float16 else _lib.DTYPE_BF16
    a.x_stride = x.stride(0)
    if logits is not None or gate_w is not None:
        if logits is not None:
            a.logits = ptr(logits)
            a.n_logits = logits.shape[1]
        else:
            a.gate_w = ptr(gate_w)
            a.n_logits = gate_w.shape[0]
        a.sel_bias = ptr(sel_bias)
        a.score_fn = SCORE_FNS[score_fn]
        a.route_scale = float(route_scale)
    a.sel = ptr(sel)
    a.weights = ptr(weights)
    a.rw_fp16 = ptr(rw)
    a.min_expert = min_expert
    a.max_expert = max_expert
    a.tables = ptr(tables)
    a.k2_per_expert = ptr(k2_per_expert)
    a.bits = float(bits) if bits is not None else 0.0
    keep = None
    if shared_ptrs is not None:
        keep = (ctypes.c_int64 * 9)(*[int(v) for v in shared_ptrs])
        a.shared = ctypes.cast(keep, ctypes.c_void_p)
        a.shared_bits = float(shared_bits)
    a.limit = float(limit)
    a.out = ptr(out)
    a.out_stride = out.stride(0) if out is not None else 0
    if residual is not None:
        a.residual = ptr(residual)
        a.residual_stride = residual.stride(0)
    if events is not None:
        a.events = ctypes.cast(events, ctypes.c_void_p)
    a.bits_down = float(bits_down) if bits_down is not None else 0.0
    a.k2_down_per_expert = ptr(k2_down_per_expert)
    a.shared_bits_down = float(shared_bits_down) if shared_bits_down is not None else 0.0
    a.shared_gate_w = ptr(shared_gate_w)
    return a, keep


def moe_forward(ws: MoeWorkspace, x: torch.Tensor, tables: torch.Tensor, out: torch.Tensor | None, *, limit: float,
                bits: float | None = None, k2_per_expert: torch.Tensor | None = None,
                logits: torch.Tensor | None = None, sel: torch.Tensor | None = None,
                weights: torch.Tensor | None = None, rw: torch.Tensor | None = None,
                score_fn: str = "sigmoid", sel_bias: torch.Tensor | None = None, route_scale: float = 1.0,
                shared_ptrs=None, shared_bits: float | None = None, min_expert: int = -1, max_expert: int = 0,
                events=None, residual: torch.Tensor | None = None, gate_w: torch.Tensor | None = None,
                bits_down: float | None = None, k2_down_per_expert: torch.Tensor | None = None,
                shared_bits_down: float | None = None, shared_gate_w: torch.Tensor | None = None):
    """One MoE layer: out[r] = sum over r's active slots (slot order) + shared expert.

    With ``logits`` the routing runs on the device and writes ``sel``/``weights``/``rw`` (all
    must be given as outputs); otherwise ``sel`` with ``weights`` (fp32) or ``rw`` (fp16) are
    the routes. ``tables``: int64 ``[9, n_local]`` device pointer table. ``shared_ptrs``: 9 ints.
    ``events``: optional ctypes array of 10 hipEvent_t handles: start and end timestamps of the
    5 stages' kernels (prepare, gate/up, activation, down, combine).
    ``residual``: optional bf16 ``[rows, H]`` stream updated in place to ``bf16(residual + bf16(y))``
    (may be ``x`` itself); ``out`` may then be None.
    ``gate_w``: optional fp32 ``[n_experts, H]`` router weight; the logits ``x @ gate_w.T`` are then
    computed on the device (instead of ``logits``) and routed with ``score_fn``/``sel_bias``.
    ``bits_down`` / ``k2_down_per_expert`` / ``shared_bits_down``: the down projections' rate when
    it differs from gate/up (the reference launcher's K_d). ``shared_gate_w``: fp16 ``[H]``; the
    shared term is then scaled by sigmoid(x . shared_gate_w) per row.
    """
    a, keep = _moe_args(ws.shape, ws.buffer.device, x, tables, out, limit, bits, k2_per_expert, logits, sel, weights,
                        rw, score_fn, sel_bias, route_scale, shared_ptrs, shared_bits, min_expert, max_expert, events,
                        residual, gate_w, bits_down, k2_down_per_expert, shared_bits_down, shared_gate_w)
    a.workspace = ptr(ws.buffer)
    a.workspace_bytes = ws.buffer.numel()
    check(lib().evamx_moe_forward(ctypes.byref(a), stream_handle(x.device)), "evamx_moe_forward")
    del keep
    return out


def moe_forward_static(shape: MoeShape, x: torch.Tensor, tables: torch.Tensor, out: torch.Tensor | None, *,
                       limit: float, bits: float | None = None, k2_per_expert: torch.Tensor | None = None,
                       logits: torch.Tensor | None = None, sel: torch.Tensor | None = None,
                       weights: torch.Tensor | None = None, rw: torch.Tensor | None = None,
                       score_fn: str = "sigmoid", sel_bias: torch.Tensor | None = None, route_scale: float = 1.0,
                       shared_ptrs=None, shared_bits: float | None = None, min_expert: int = -1,
                       max_expert: int = 0, events=None, residual: torch.Tensor | None = None,
                       gate_w: torch.Tensor | None = None, bits_down: float | None = None,
                       k2_down_per_expert: torch.Tensor | None = None, shared_bits_down: float | None = None,
                       shared_gate_w: torch.Tensor | None = None):
    """``moe_forward`` without a workspace: evamx_moe_forward_static runs the layer on the
    library's fixed device scratch (64 MiB per GPU) and allocates nothing, for callers that
    cannot allocate (e.g. under graph capture). ``shape`` is the MoeShape a workspace would have
    been built for. Calls that overlap on one GPU share the scratch and race."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError("x must be a device tensor")
    a, keep = _moe_args(shape, x.device, x, tables, out, limit, bits, k2_per_expert, logits, sel, weights, rw,
                        score_fn, sel_bias, route_scale, shared_ptrs, shared_bits, min_expert, max_expert, events,
                        residual, gate_w, bits_down, k2_down_per_expert, shared_bits_down, shared_gate_w)
    check(lib().evamx_moe_forward_static(ctypes.byref(a), stream_handle(x.device)), "evamx_moe_forward_static")
    del keep
    return out


def w4_moe_forward(x: torch.Tensor, gate: W4Weight, up: W4Weight, down: W4Weight, sel: torch.Tensor, weights: torch.Tensor, *,
                   n_shared: int = 0, first_expert: int = 0, limit: float = 0.0, out: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """One MoE layer's experts on 4-bit weights with group scales, for given routes: ``x`` fp16 or bf16
    ``[rows, hidden]``, ``sel`` int64 and ``weights`` fp32 ``[rows, topk]`` (``route`` / ``route_topk``), the
    result of x's dtype. ``gate`` and ``up`` are stacks ``[inter, hidden]``, ``down`` ``[hidden, inter]``: the
    experts ``first_expert`` and up, then ``n_shared`` shared experts that every token takes with weight 1.
    Slots of other experts add nothing (expert parallelism). ``limit`` clamps as in ``moe_forward``, but a
    NaN stays NaN (a routed expert there takes it to the limit). ``out`` must not overlap ``x``. At most 65536 slots, 2^31 padded values of ``x`` and 2^30 hidden activations a
    call (``W4Experts`` splits larger ones)."""
    x_stride = _row_stride(x, "x")
    if x.dtype not in _DTYPES:
        raise ValueError("x must be fp16 or bf16")
    rows, hidden = x.shape
    _dev(sel, "sel", torch.int64, 2)
    _dev(weights, "weights", torch.float32, 2)
    if sel.shape[0] != rows or weights.shape != sel.shape:
        raise ValueError(f"sel {tuple(sel.shape)} and weights {tuple(weights.shape)} must be [{rows}, topk]")
    if gate.n_in != hidden:
        raise ValueError(f"x has {hidden} features, the experts {gate.n_in}")
    if out is None:
        out = torch.empty(rows, hidden, dtype=x.dtype, device=x.device)
    out_stride = _row_stride(out, "out", x.dtype)
    if tuple(out.shape) != (rows, hidden):
        raise ValueError(f"out must be [{rows}, {hidden}]")
    _no_grad("w4_moe_forward", x, weights, out)
    if workspace is None:
        need = lib().evamx_w4_moe_workspace_bytes(rows, sel.shape[1], n_shared, hidden, gate.n_out)
        if need == 0:
            raise ValueError(lib().evamx_last_error().decode())
        workspace = torch.empty(need, dtype=torch.uint8, device=x.device)
    _dev(workspace, "workspace", torch.uint8, 1)
    for t, name in ((sel, "sel"), (weights, "weights"), (gate, "gate"), (up, "up"), (down, "down"), (out, "out"), (workspace, "workspace")):
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
    a = W4MoeArgs(ptr(x), ptr(sel), ptr(weights), ctypes.pointer(gate.desc), ctypes.pointer(up.desc), ctypes.pointer(down.desc), ptr(out),
                  ptr(workspace), workspace.numel(), x_stride, out_stride, first_expert, _DTYPES[x.dtype], rows, sel.shape[1], n_shared,
                  float(limit))
    _launch(lib().evamx_w4_moe_forward, "evamx_w4_moe_forward", x.device, ctypes.byref(a))
    return out


def read_floor(ncg: int, rows: int, waves: int, device=None, reps: int = 50) -> float:
    """Bytes per second of the read-only benchmark (evamx_bench_read): ``waves`` waves stream
    ``rows`` 1 KiB chunks each in a decode GEMV launch's shape (wave w reads column group w % ncg
    of its chain's rows), no decode; ``reps`` back-to-back launches timed with events. The
    launches cycle through distinct copies totalling at least 1 GiB, as the layer benchmark
    cycles its weights, so that the 256 MiB Infinity Cache cannot serve a repeated buffer."""
    dev = torch.device("cuda", 0) if device is None else torch.device(device)
    nbytes = (waves // ncg) * rows * ncg * 1024
    copies = min(64, max(2, -(-(1 << 30) // nbytes)))
    buf = torch.zeros(copies * nbytes, dtype=torch.uint8, device=dev)
    sink = torch.zeros(64, dtype=torch.float32, device=dev)
    stream = stream_handle(dev)
    base = ptr(buf)

    def launch(i):
        check(lib().evamx_bench_read(base + (i % copies) * nbytes, nbytes, ncg, rows, waves, ptr(sink), stream),
              "evamx_bench_read")

    for i in range(copies):   # warm-up: every copy once
        launch(i)
    e0 = torch.cuda.Event(enable_timing=True)
    e1 = torch.cuda.Event(enable_timing=True)
    e0.record()
    for i in range(reps):
        launch(i)
    e1.record()
    e1.synchronize()
    return nbytes * reps / (e0.elapsed_time(e1) * 1e-3)


def decode_ceiling(bits: float, device=None, waves: int | None = None, iters: int = 4000) -> float:
    """Decoded weights per second of the register-only decode benchmark (evamx_bench_decode):
    the arithmetic bound of the decode GEMV at ``bits``, timed with events on the current stream."""
    dev = torch.device("cuda", 0) if device is None else torch.device(device)
    if waves is None:
        waves = torch.cuda.get_device_properties(dev).multi_processor_count * 16
    sink = torch.zeros(256, dtype=torch.float32, device=dev)
    stream = stream_handle(dev)
    check(lib().evamx_bench_decode(float(bits), waves, 16, ptr(sink), stream), "evamx_bench_decode")   # warm-up
    e0 = torch.cuda.Event(enable_timing=True)
    e1 = torch.cuda.Event(enable_timing=True)
    e0.record()
    check(lib().evamx_bench_decode(float(bits), waves, iters, ptr(sink), stream), "evamx_bench_decode")
    e1.record()
    e1.synchronize()
    return waves * 64.0 * 32.0 * iters / (e0.elapsed_time(e1) * 1e-3)
