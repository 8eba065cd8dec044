"""The operators of a mixture-of-experts layer on 16-bit weights, forward and backward: what is measured, in
which sizes, and their plain forms.

Kinds of case:

- ``sort``      ``ops.expert_order`` and ``ops.sort_tokens``: tokens sorted by expert, and the tokens' gradient;
- ``combine``   ``ops.combine_tokens``: sorted rows back to their tokens with weights, and both gradients;
- ``linear``    ``ops.linear``: ``act(x W^T + bias) + residual``, and the gradients of x, W and bias;
- ``experts``   ``ops.expert_linear``: the same for sorted rows, each expert's with its own matrix.
"""
import functools
import math

import torch

own = False


def _sort(name, rows, **kw):
    case = {"name": name, "kind": "sort", "rows": rows, "hidden": 7168, "experts": 256, "topk": 8, "first": 0, "local": 256,
            "padded": False, "routing": "normal", "dtype": "bf16", "train": False}
    case.update(kw)
    return case


def _combine(name, rows, **kw):
    case = {"name": name, "kind": "combine", "rows": rows, "hidden": 7168, "experts": 256, "topk": 8, "first": 0, "local": 256,
            "padded": False, "routing": "normal", "dtype": "bf16", "residual": False, "train": False}
    case.update(kw)
    return case


def _linear(name, rows, n_in, n_out, **kw):
    case = {"name": name, "kind": "linear", "rows": rows, "in": n_in, "out": n_out, "bias": False, "act": "none", "limit": 0.0,
            "residual": False, "dtype": "bf16", "train": False}
    case.update(kw)
    return case


def _experts(name, rows, n_in, n_out, **kw):
    case = {"name": name, "kind": "experts", "rows": rows, "in": n_in, "out": n_out, "experts": 256, "topk": 8, "first": 0,
            "local": 256, "padded": False, "routing": "normal", "bias": False, "act": "none", "limit": 0.0, "dtype": "bf16",
            "train": False}
    case.update(kw)
    return case


def listed():
    return [
        # one decoded token in front of the experts: launch and latency
        _sort("sort_1", 1),
        # one rank's quarter of the experts for a padded batch gathered from all ranks, fine-tuned
        _sort("sort_ep_3001_train", 3001, hidden=5120, experts=384, topk=6, first=192, local=96, padded=True, dtype="fp16", train=True),
        # a long training batch with hot experts
        _sort("sort_16384_train", 16384, routing="skewed", train=True),
        # a decode batch behind the experts, added to the residual stream
        _combine("combine_16", 16, residual=True),
        # a training batch behind the experts
        _combine("combine_8191_train", 8191, train=True),
        # one decoded token through a layer's output projection
        _linear("linear_1", 1, 2048, 7168, residual=True),
        # a decode batch through a projection whose sizes are no multiple of anything
        _linear("linear_13_odd", 13, 5001, 2303, bias=True, act="gelu", residual=True, dtype="fp16"),
        # a long prompt through a dense layer's gate and up products
        _linear("linear_8192_swiglu", 8192, 7168, 4096, act="swiglu"),
        # a fine-tuning step of a projection on a short batch
        _linear("linear_2000_train", 2000, 2048, 5120, bias=True, act="silu", train=True),
        # a decode batch at one rank's quarter of the experts: their weights are what is read
        _experts("experts_16", 16, 7168, 4096, first=64, local=64, act="swiglu", limit=10.0),
        # a prefill chunk at one rank's quarter of the experts, Zipf loads: the down products
        _experts("experts_6000_down", 6000, 2048, 7168, local=64, routing="zipf", dtype="fp16"),
        # a training batch at one rank's eighth of the experts: gate and up products, all gradients
        _experts("experts_4096_train", 4096, 7168, 4096, first=32, local=32, act="swiglu", train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


LAYERS = [(7168, 2048, 256, 8), (5120, 2304, 384, 6), (4096, 1536, 128, 8), (2048, 768, 64, 6), (1024, 512, 16, 4), (640, 384, 40, 3),
          (1000, 333, 24, 5), (2048, 512, 8, 1)]


def draw(rng):
    kind = rng.choice(["sort", "combine", "linear", "linear", "experts", "experts"])
    train, dtype, routing = rng.random() < 0.5, rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["normal", "skewed", "zipf"])
    hidden, inter, experts, topk = rng.choice(LAYERS)
    local = experts if rng.random() < 0.5 else rng.randint(1, experts)
    ep = {"experts": experts, "topk": topk, "first": rng.randint(0, experts - local), "local": local, "padded": rng.random() < 0.3,
          "routing": routing, "dtype": dtype, "train": train}
    if kind in ("sort", "combine"):
        if rng.random() < 0.2:
            ep["dtype"] = "fp32"
        rows = _log_int(rng, 1, min(8000, 450_000_000 // (hidden * topk)))
        case = _sort("", rows, hidden=hidden, **ep) if kind == "sort" else _combine("", rows, hidden=hidden, residual=rng.random() < 0.5, **ep)
    else:
        act = rng.choice(["none", "none", "silu", "gelu", "relu", "swiglu", "swiglu"])
        kw = {"act": act, "limit": rng.choice([0.0, 10.0]) if act == "swiglu" else 0.0, "bias": rng.random() < 0.4}
        if kind == "linear":
            n_in, n_out = _log_int(rng, 64, 9000), _log_int(rng, 64, 9000)
            if rng.random() < 0.7:
                n_in, n_out = -(-n_in // 64) * 64, -(-n_out // 64) * 64
            n_out += n_out % 2 if act == "swiglu" else 0
            case = _linear("", _log_int(rng, 1, 3000), n_in, n_out, residual=not train and rng.random() < 0.4, dtype=dtype, train=train, **kw)
        else:
            n_in, n_out = (hidden, 2 * inter) if rng.random() < 0.6 or act == "swiglu" else (inter, hidden)
            most = 300_000_000 // (n_in * n_out)            # matrices: about 600 MB of them
            if local > most:
                ep["local"] = most
            case = _experts("", _log_int(rng, 1, 1500), n_in, n_out, **ep, **kw)
    del case["name"]
    return case


# ---- inputs -----------------------------------------------------------------------------------

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _routes(g, case):
    """Experts that the rows pick, int64 ``[rows, topk]``; the padding's rows pick none (-1)."""
    rows, experts, topk, routing = case["rows"], case["experts"], case["topk"], case["routing"]
    z = torch.randn(rows, experts, generator=g, device="cuda")
    order = torch.randperm(experts, generator=g, device="cuda")
    if routing == "skewed":      # two experts that every token picks
        z[:, order[:2]] += 6.0
    elif routing == "zipf":      # picks without replacement, Zipf(1.1) over the experts
        u = torch.rand(rows, experts, generator=g, device="cuda", dtype=torch.float64).clamp_(1e-300, 1.0)
        z = -1.1 * torch.log(torch.arange(1, experts + 1, dtype=torch.float64, device="cuda"))[order] - torch.log(-torch.log(u))
    sel = z.topk(topk, dim=1).indices
    if case["padded"]:
        sel[torch.rand(rows, generator=g, device="cuda") < 0.1] = -1
    return sel.contiguous()


def _order(sel, first, local):
    """``starts`` int32 ``[local + 1]`` of the local experts' rows and ``position`` int32 ``[rows, topk]``, each
    slot's row (-1: another rank's expert, or none): rows by expert, an expert's in the order of the slots."""
    expert = (sel - first).flatten()
    expert = torch.where((expert >= 0) & (expert < local), expert, local)
    by = expert.argsort(stable=True)
    position = torch.empty_like(by)
    position[by] = torch.arange(by.numel(), device=by.device)
    position = torch.where(expert < local, position, -1).to(torch.int32).view(sel.shape)
    starts = torch.searchsorted(expert[by], torch.arange(local + 1, device=by.device)).to(torch.int32)
    return starts, position


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale).to(dtype)

    s = {"kind": case["kind"], "train": case["train"]}
    if case["kind"] != "linear":
        s["sel"] = _routes(g, case)
        s["first"], s["local"] = case["first"], case["local"]
    slots = case["rows"] * case.get("topk", 1)
    if case["kind"] == "sort":
        s["x"] = randn(case["rows"], case["hidden"])
        s["grad"] = randn(slots, case["hidden"]) if case["train"] else None
    elif case["kind"] == "combine":
        s["starts"], s["position"] = _order(s.pop("sel"), case["first"], case["local"])
        s["y"] = randn(slots, case["hidden"])
        w = torch.rand(case["rows"], case["topk"], generator=g, device="cuda") + 0.05
        s["weights"] = w / w.sum(1, keepdim=True)
        s["residual"] = randn(case["rows"], case["hidden"]) if case["residual"] else None
        s["grad"] = randn(case["rows"], case["hidden"]) if case["train"] else None
    else:
        stack, rows = ((), case["rows"]) if case["kind"] == "linear" else ((case["local"],), slots)
        if stack:
            s["starts"], _ = _order(s.pop("sel"), case["first"], case["local"])
        s["x"] = randn(rows, case["in"])
        s["w"] = randn(*stack, case["out"], case["in"], scale=1.5 * case["in"] ** -0.5)
        s["bias"] = randn(*stack, case["out"]) if case["bias"] else None
        y_cols = case["out"] // 2 if case["act"] == "swiglu" else case["out"]
        s["residual"] = randn(rows, y_cols) if case.get("residual") else None
        s["grad"] = randn(rows, y_cols) if case["train"] else None
        s["act"], s["limit"] = case["act"], case["limit"]
    return s


# ---- one pass ---------------------------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    return {"sort": _plain_sort, "combine": _plain_combine, "linear": _plain_product, "experts": _plain_product}[s["kind"]](s)


def _run_own(s):
    from eva_amd import ops

    train = s["train"]
    leaf = (lambda t: None if t is None else t.detach().requires_grad_()) if train else (lambda t: t)
    if s["kind"] == "sort":
        x = leaf(s["x"])
        order = ops.expert_order(s["sel"], s["local"], first_expert=s["first"])
        rows = ops.sort_tokens(x, order)
        out = {"starts": order.starts, "position": order.position, "rows": rows.detach()}
        if train:
            out["dx"], = torch.autograd.grad(rows, x, s["grad"])
        return out
    if s["kind"] == "combine":
        y, weights = leaf(s["y"]), leaf(s["weights"])
        out = ops.combine_tokens(y, ops.ExpertOrder(s["starts"], s["position"]), weights, residual=s["residual"])
        if not train:
            return out
        dy, dweights = torch.autograd.grad(out, (y, weights), s["grad"])
        return {"out": out.detach(), "dy": dy, "dweights": dweights}
    x, w, bias = leaf(s["x"]), leaf(s["w"]), leaf(s["bias"])
    act = None if s["act"] == "none" else s["act"]
    if s["kind"] == "linear":
        y = ops.linear(x, w, bias, activation=act, limit=s["limit"], residual=s["residual"])
    else:
        y = ops.expert_linear(x, w, s["starts"], bias, activation=act, limit=s["limit"])
    if not train:
        return y
    grads = torch.autograd.grad(y, (x, w) if bias is None else (x, w, bias), s["grad"])
    return {"y": y.detach(), **dict(zip(("dx", "dw", "dbias"), grads))}


def _plain_sort(s):
    starts, position = _order(s["sel"], s["first"], s["local"])
    token, k = (position >= 0).nonzero(as_tuple=True)
    rows = s["x"].new_zeros(position.numel(), s["x"].shape[1])
    rows[position[token, k].long()] = s["x"][token]
    out = {"starts": starts, "position": position, "rows": rows}
    if s["train"]:
        g = s["grad"][position.clamp(min=0).long()].float()
        out["dx"] = torch.where((position >= 0)[..., None], g, 0.0).sum(1).to(s["x"].dtype)
    return out


def _plain_combine(s):
    position, here, w = s["position"].clamp(min=0).long(), s["position"] >= 0, s["weights"]
    y = torch.where(here[..., None], s["y"][position].float(), 0.0)
    out = (w[..., None] * y).sum(1)
    out = (out if s["residual"] is None else out + s["residual"].float()).to(s["y"].dtype)
    if not s["train"]:
        return out
    g = s["grad"].float()
    dw = torch.where(here, (g[:, None] * y).sum(2), 0.0)
    dy = torch.zeros_like(s["y"])
    token, k = here.nonzero(as_tuple=True)
    dy[position[token, k]] = (w[token, k, None] * g[token]).to(dy.dtype)
    return {"out": out, "dy": dy, "dweights": dw}


def _act(pre, act, limit):
    """The activation of ``pre`` and, of a grad in its result, the grad in ``pre``."""
    if act == "none":
        return pre, lambda g: g
    if act == "relu":
        return torch.where(pre > 0, pre, 0.0), lambda g: torch.where(pre > 0, g, 0.0)
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(pre * 0.5 ** 0.5))
        return pre * cdf, lambda g: g * (cdf + pre * torch.exp(-0.5 * pre * pre) * (2 * math.pi) ** -0.5)
    gate, up = (pre, None) if act == "silu" else pre.chunk(2, -1)
    sigma = 1 / (1 + torch.exp(-gate))
    silu, slope = gate * sigma, sigma * (1 + gate * (1 - sigma))
    if act == "silu":
        return silu, lambda g: g * slope
    if limit == 0:
        return silu * up, lambda g: torch.cat((g * up * slope, g * silu), -1)
    a, u = silu.clamp(max=limit), up.clamp(-limit, limit)
    return a * u, lambda g: torch.cat((torch.where(silu <= limit, g * u * slope, 0.0), torch.where(up.abs() <= limit, g * a, 0.0)), -1)


def _plain_product(s):
    x, w, starts = s["x"].float(), s["w"], s.get("starts")
    if starts is None:
        at, used, w = None, None, w.float()
    else:                        # the experts that have rows, each one's padded to the most of any
        local, every = w.shape[0], x.shape[0]
        expert = torch.searchsorted(starts[1:].contiguous(), torch.arange(every, device=x.device, dtype=torch.int32), right=True)
        row, = (expert < local).nonzero(as_tuple=True)
        expert = expert[row]
        used, unit = expert.unique(return_inverse=True)
        place = row - starts.long()[expert]
        most = int(place.max()) + 1 if row.numel() else 0
        at = (unit, place)
        w = w[used].float()

        def spread(t):
            a = t.new_zeros(used.numel(), most, t.shape[1])
            a[at] = t[row]
            return a

        def collect(t):
            a = t.new_zeros(every, t.shape[2])
            a[row] = t[at]
            return a

        x = spread(x)
    bias = None if s["bias"] is None else s["bias"].float() if at is None else s["bias"][used].float()[:, None]
    pre = x @ w.transpose(-1, -2)
    y, back = _act(pre if bias is None else pre + bias, s["act"], s["limit"])
    y = y if at is None else collect(y)
    y = (y if s["residual"] is None else y + s["residual"].float()).to(s["x"].dtype)
    if not s["train"]:
        return y
    g = back(s["grad"].float() if at is None else spread(s["grad"].float()))
    dx, dw, db = g @ w, g.transpose(-1, -2) @ x, g.sum(-2)
    if at is not None:
        dx = collect(dx)
        dw = s["w"].new_zeros(s["w"].shape).index_copy_(0, used, dw.to(s["w"].dtype))
        db = db.new_zeros(local, db.shape[1]).index_copy_(0, used, db)
    out = {"y": y, "dx": dx.to(s["x"].dtype), "dw": dw.to(s["w"].dtype)}
    if s["bias"] is not None:
        out["dbias"] = db.to(s["w"].dtype)
    return out


# ---- what a pass cannot do without ------------------------------------------------------------


@functools.lru_cache(maxsize=None)
def _touched(rows, experts, topk, routing, first, local, padded):
    """Local experts that at least one of the rows picks, and the rows' picks of them, as one draw of this routing has it."""
    g = torch.Generator()
    g.manual_seed(1)
    z = torch.randn(rows, experts, generator=g)
    order = torch.randperm(experts, generator=g)
    if routing == "skewed":
        z[:, order[:2]] += 6.0
    elif routing == "zipf":
        z = -1.1 * torch.log(order + 1.0) - torch.log(-torch.log(torch.rand(rows, experts, generator=g)))
    sel = z.topk(topk, dim=1).indices
    if padded:
        sel = sel[torch.rand(rows, generator=g) >= 0.1]
    sel = sel[(sel >= first) & (sel < first + local)]
    return int(sel.unique().numel()), int(sel.numel())


def work(case):
    rows, item, train = case["rows"], 4 if case["dtype"] == "fp32" else 2, case["train"]
    if case["kind"] != "linear":
        used, slots = _touched(*(case[k] for k in ("rows", "experts", "topk", "routing", "first", "local", "padded")))
        every = rows * case["topk"]                  # rows of the sorted tensors, the empty ones behind the last among them
    if case["kind"] == "sort":
        h = item * case["hidden"]
        return {"bytes": 12 * every + 4 * case["local"] + h * (rows + every) + (h * (slots + rows) if train else 0),
                "flops": float(slots * case["hidden"]) if train else 0.0}
    if case["kind"] == "combine":
        h = item * case["hidden"]
        back = h * (rows + every) + 4 * every if train else 0    # y and the weights are read for the forward already
        return {"bytes": 8 * every + h * (slots + rows * (2 if case["residual"] else 1)) + back,
                "flops": (5.0 if train else 2.0) * slots * case["hidden"]}
    a, b = case["in"], case["out"]
    y = b // 2 if case["act"] == "swiglu" else b
    if case["kind"] == "linear":
        used = mats = 1
        slots = every = rows
    else:
        mats = case["local"]
    read = used * a * b + slots * a + (used * b if case["bias"] else 0) + (every * y if case.get("residual") else 0)
    back = slots * y + every * a + mats * a * b + (mats * b if case["bias"] else 0)
    return {"bytes": item * (read + every * y + (back if train else 0)), "flops": (6.0 if train else 2.0) * slots * a * b}


# ---- the same results in 64 bits --------------------------------------------------------------


def _exact_act(pre, act, limit):
    if act in ("none", "relu", "gelu"):
        return pre if act == "none" else torch.relu(pre) if act == "relu" else pre * torch.special.ndtr(pre)
    if act == "silu":
        return pre * torch.sigmoid(pre)
    half = pre.shape[1] // 2
    a, u = pre[:, :half] * torch.sigmoid(pre[:, :half]), pre[:, half:]
    if limit:
        a, u = torch.minimum(a, a.new_tensor(limit)), torch.maximum(torch.minimum(u, u.new_tensor(limit)), u.new_tensor(-limit))
    return a * u


def exact(case, seed):
    s = prepare(case, seed)
    train = case["train"]
    if case["kind"] == "sort":
        lists = [[] for _ in range(case["local"])]
        for slot, e in enumerate(s["sel"].flatten().tolist()):
            if 0 <= e - case["first"] < case["local"]:
                lists[e - case["first"]].append(slot)
        slots = torch.tensor([v for part in lists for v in part], dtype=torch.int64, device="cuda")
        token, n = slots // case["topk"], slots.numel()
        rows = torch.zeros(s["sel"].numel(), case["hidden"], dtype=torch.float64, device="cuda")
        rows[:n] = s["x"][token].double()
        out = {"starts": None, "position": None, "rows": rows}
        if train:
            out["dx"] = torch.zeros(case["rows"], case["hidden"], dtype=torch.float64, device="cuda").index_add_(0, token, s["grad"][:n].double())
        return out
    if case["kind"] == "combine":
        out = torch.zeros(case["rows"], case["hidden"], dtype=torch.float64, device="cuda") if s["residual"] is None else s["residual"].double()
        dw = torch.zeros(case["rows"], case["topk"], dtype=torch.float64, device="cuda")
        dy = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda") if train else None
        for k in range(case["topk"]):
            token, = (s["position"][:, k] >= 0).nonzero(as_tuple=True)
            row = s["position"][token, k].long()
            y, w = s["y"][row].double(), s["weights"][token, k, None].double()
            out[token] += w * y
            if train:
                g = s["grad"][token].double()
                dy[row], dw[token, k] = w * g, (g * y).sum(1)
        return {"out": out, "dy": dy, "dweights": dw} if train else out
    starts = [0, case["rows"]] if case["kind"] == "linear" else s["starts"].tolist()
    w, bias = (t if t is None or case["kind"] == "experts" else t[None] for t in (s["w"], s["bias"]))
    cols = case["out"] // 2 if case["act"] == "swiglu" else case["out"]
    y = torch.zeros(s["x"].shape[0], cols, dtype=torch.float64, device="cuda")
    dx, dw = (torch.zeros(t.shape, dtype=torch.float64, device="cuda") if train else None for t in (s["x"], w))
    db = torch.zeros(len(starts) - 1, case["out"], dtype=torch.float64, device="cuda")
    for e, (lo, hi) in enumerate(zip(starts[:-1], starts[1:])):
        if lo == hi:
            continue
        x, m = s["x"][lo:hi].double(), w[e].double()
        pre = x @ m.t()
        if bias is not None:
            pre += bias[e].double()
        pre.requires_grad_(train)
        part = _exact_act(pre, case["act"], case["limit"])
        y[lo:hi] = part.detach()
        if train:
            d, = torch.autograd.grad(part, pre, s["grad"][lo:hi].double()) if case["act"] != "none" else (s["grad"][lo:hi].double(),)
            dx[lo:hi], dw[e], db[e] = d @ m, d.t() @ x, d.sum(0)
    if s["residual"] is not None:
        y += s["residual"].double()
    if not train:
        return y
    out = {"y": y, "dx": dx, "dw": dw if case["kind"] == "experts" else dw[0]}
    if bias is not None:
        out["dbias"] = db if case["kind"] == "experts" else db[0]
    return out
