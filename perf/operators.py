"""Cases for timing the dense tail of a training step: dropout from the counter generator, layer norm with its residual, and the
class head whose logits are never kept. `run` computes each either in its plain form (elementary torch operations in 32 bits, rounded
once at the end) or, where `own` is true, through pagraph_amd's entry points as a user calls them."""
import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_M32 = 0xFFFFFFFF


def listed():
    return [
        # one vertex's hidden row on its own: what a call costs
        {"name": "dropout-one-row", "op": "dropout", "n": 1, "d": 64, "type": "fp32", "p": 0.2, "train": False},
        # a batch of raw feature rows (batch 6000, Reddit's 602 columns: rows that are no whole number of 16-byte pieces)
        {"name": "dropout-features", "op": "dropout", "n": 6000, "d": 602, "type": "fp32", "p": 0.2, "train": True},
        # a long batch of wide rows in 16 bits
        {"name": "dropout-wide", "op": "dropout", "n": 16384, "d": 2048, "type": "bf16", "p": 0.5, "train": True},
        # one row while answering
        {"name": "norm-one-row", "op": "norm", "n": 1, "d": 1024, "type": "bf16", "p": 0.0, "residual": False, "train": False},
        # the hidden rows of a minibatch's first layer (2 x 32 hidden units behind the skip-concat), a training step
        {"name": "norm-hidden", "op": "norm", "n": 12000, "d": 64, "type": "fp32", "p": 0.0, "residual": False, "train": True},
        # raw feature rows with the residual, Reddit's odd width
        {"name": "norm-features", "op": "norm", "n": 6000, "d": 602, "type": "fp32", "p": 0.0, "residual": True, "train": True},
        # a residual block's end on wide rows: dropout, residual sum and norm, with every gradient
        {"name": "norm-block", "op": "norm", "n": 16384, "d": 2048, "type": "bf16", "p": 0.1, "residual": True, "train": True},
        # one row against a class table while answering: the table is read once
        {"name": "loss-one-row", "op": "loss", "n": 1, "k": 64, "c": 1000, "type": "fp32", "ignored": 0.0, "train": False},
        # a half-precision head with nothing even about it
        {"name": "loss-odd", "op": "loss", "n": 777, "k": 602, "c": 1153, "type": "fp16", "ignored": 0.1, "train": True},
        # evaluation over a held-out batch: every row's loss, no gradient
        {"name": "loss-score", "op": "loss", "n": 4096, "k": 256, "c": 32000, "type": "bf16", "ignored": 0.0, "train": False},
        # the sampled GCN's head (batch 6000, 2 x 32 hidden columns) over a large label set, a training step in the models' own type
        {"name": "loss-gcn", "op": "loss", "n": 6000, "k": 64, "c": 50000, "type": "fp32", "ignored": 0.05, "train": True},
        # a wide head in 16 bits, a training step
        {"name": "loss-wide", "op": "loss", "n": 8192, "k": 1024, "c": 65536, "type": "bf16", "ignored": 0.05, "train": True},
    ]


def _log(rng, lo, hi):
    v = int(round(lo * (hi / lo) ** rng.random()))
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["dropout", "norm", "loss", "loss"])
    dt = rng.choice(["fp32", "bf16", "fp16"])
    train = rng.random() < 0.75
    if op == "loss":
        while True:
            n, k, c = _log(rng, 1, 16384), _log(rng, 16, 1024), _log(rng, 61, 131072)
            if n * k * c <= 2 ** 36 * (0.25 if dt == "fp32" else 1.0) and n * c <= 2 ** 29:
                return {"op": "loss", "n": n, "k": k, "c": c, "type": dt, "ignored": rng.choice([0.0, 0.05, 0.3]), "train": train}
    while True:
        n, d = _log(rng, 1, 65536), _log(rng, 16, 8192)
        if n * d <= 2 ** 24:
            break
    case = {"op": op, "n": n, "d": d, "type": dt, "p": rng.choice([0.1, 0.2, 0.5]), "train": train}
    if op == "norm":
        case["residual"] = rng.random() < 0.5
        if not case["residual"] or rng.random() < 0.5:
            case["p"] = 0.0
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------------------
def _inputs(case, seed, dev):
    """the case's tensors on `dev`, drawn there from the seed alone"""
    g = torch.Generator(device=dev)
    g.manual_seed(seed * 7919 + 17)
    t = _TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale + shift).to(t)

    if case["op"] == "loss":
        n, k, c = case["n"], case["k"], case["c"]
        labels = (torch.rand(n, generator=g, device=dev) ** 2 * c).long().clamp_(0, c - 1)      # some classes are common
        skip = torch.rand(n, generator=g, device=dev) < case["ignored"]
        skip[0] = False
        return {"h": normal(n, k), "w": normal(c, k, scale=2.0 / k ** 0.5), "b": normal(c, scale=0.5),
                "labels": torch.where(skip, torch.full_like(labels, -100), labels)}
    n, d = case["n"], case["d"]
    out = {"x": normal(n, d, scale=1.5, shift=0.25)}
    if case["op"] == "norm":
        out["w"], out["b"] = normal(d, scale=0.25, shift=1.0), normal(d, scale=0.25)
        if case["residual"]:
            out["res"] = normal(n, d)
            if case["train"]:
                out["gs"] = normal(n, d, scale=0.1)
    if case["train"]:
        out["gy"] = normal(n, d, scale=0.1)
    return out


def _mask_key(case, seed):
    """(threshold, seed, tag, step) of the case's mask; None without dropout"""
    if case.get("p", 0.0) == 0.0:
        return None
    return int(round(case["p"] * 65536.0)), (seed * 0x9E3779B97F4A7C15 + 5) & 0xFFFFFFFFFFFFFFFF, 3, seed % 1000 + 1


def prepare(case, seed):
    dev = torch.device("cuda")
    t = _inputs(case, seed, dev)
    state = {"case": case}
    leaf = lambda x: x.requires_grad_(case["train"])
    if case["op"] == "loss":
        lin = torch.nn.Linear(case["k"], case["c"], device=dev, dtype=t["h"].dtype)
        with torch.no_grad():
            lin.weight.copy_(t["w"]), lin.bias.copy_(t["b"])
        lin.requires_grad_(case["train"])
        return {**state, "h": leaf(t["h"]), "lin": lin, "labels": t["labels"]}
    state["x"] = leaf(t["x"])
    if case["op"] == "norm":
        norm = torch.nn.LayerNorm(case["d"], device=dev, dtype=t["x"].dtype)
        with torch.no_grad():
            norm.weight.copy_(t["w"]), norm.bias.copy_(t["b"])
        norm.requires_grad_(case["train"])
        state["norm"] = norm
        if "res" in t:
            state["res"] = leaf(t["res"])
    key = _mask_key(case, seed)
    if key is not None:
        state["key"] = key
        state["step"] = torch.tensor([key[3]], dtype=torch.int64, device=dev)
    return {**state, **{name: t[name] for name in ("gy", "gs") if name in t}}


# ---- the plain forms -------------------------------------------------------------------------------------------------------
def _philox(c0, c1, c2, c3, k0, k1):
    """Philox4x32-10 on int64 tensors that hold 32-bit words"""
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57          # the low 64 bits of the product are the ones wanted
        c0, c1, c2, c3 = ((p1 >> 32) & _M32) ^ c1 ^ k0, p1 & _M32, ((p0 >> 32) & _M32) ^ c3 ^ k1, p0 & _M32
        k0, k1 = (k0 + 0x9E3779B9) & _M32, (k1 + 0xBB67AE85) & _M32
    return c0, c1, c2, c3


def _keep_scale(n, d, key, step, dev):
    """the mask of pg_dropout_t times the scale of what is kept, [n, d] in 32 bits"""
    thr, seed, tag, _ = key
    piece = torch.arange((d + 3) // 4, device=dev)
    q = (piece // 128) * 64 + piece % 64
    width = int(((d + 3) // 4 + 127) // 128 * 64)           # counters 0 .. width-1 cover every q
    r = torch.arange(n, device=dev).view(n, 1)
    uq = torch.arange(width, device=dev).view(1, width)
    zero = torch.zeros_like(r + uq)
    w = _philox(r + zero, uq + zero, zero + tag, zero + (step.view(1, 1) & _M32), seed & _M32, seed >> 32)
    w = torch.stack(w, dim=2)[:, q, :]                      # [n, pieces, 4 words]
    half = ((piece // 64) % 2).view(1, -1, 1)
    w = torch.where(half == 1, w[:, :, 2:], w[:, :, :2])    # the piece's two words
    u16 = torch.stack((w & 0xFFFF, w >> 16), dim=3).reshape(n, -1)[:, :d]
    return (u16 >= thr).float() * (65536.0 / (65536 - thr))


def _plain_dropout(s):
    x = s["x"].detach()
    ks = _keep_scale(x.size(0), x.size(1), s["key"], s["step"], x.device)
    out = {"y": (x.float() * ks).to(x.dtype)}
    if s["case"]["train"]:
        out["dx"] = (s["gy"].float() * ks).to(x.dtype)
    return out


def _plain_norm(s):
    x, t = s["x"].detach(), s["x"].dtype
    w, b = s["norm"].weight.detach().float(), s["norm"].bias.detach().float()
    ks = _keep_scale(x.size(0), x.size(1), s["key"], s["step"], x.device) if "key" in s else None
    v = x.float() if ks is None else x.float() * ks
    out = {}
    if "res" in s:
        out["s"] = (v + s["res"].detach().float()).to(t)
        v = out["s"].float()                                # what the block hands on is what is normalised
    centred = v - v.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(dim=1, keepdim=True) + s["norm"].eps)
    xh = centred * rstd
    out["y"] = (xh * w + b).to(t)
    if not s["case"]["train"]:
        return out
    gy = s["gy"].float()
    gh = gy * w
    ds = rstd * (gh - gh.mean(dim=1, keepdim=True) - xh * (gh * xh).mean(dim=1, keepdim=True))
    if "res" in s:
        ds = ds + s["gs"].float()
        out["dres"] = ds.to(t)
    out["dx"] = (ds if ks is None else ds * ks).to(t)
    out["dw"], out["db"] = (gy * xh).sum(dim=0).to(t), gy.sum(dim=0).to(t)
    return out


def _plain_loss(s):
    h, w, b, lab = s["h"].detach(), s["lin"].weight.detach(), s["lin"].bias.detach(), s["labels"]
    h32, w32 = h.float(), w.float()
    z = h32 @ w32.t() + b.float()
    top = z.max(dim=1, keepdim=True).values
    lse = top + torch.log(torch.exp(z - top).sum(dim=1, keepdim=True))
    valid = ((lab >= 0) & (lab < z.size(1))).float().view(-1, 1)
    at = lab.clamp(0, z.size(1) - 1).view(-1, 1)
    each = (lse - z.gather(1, at)) * valid
    if not s["case"]["train"]:
        return {"loss": each.view(-1)}
    count = valid.sum()
    out = {"loss": each.sum() / count}
    g = torch.exp(z - lse)
    g.scatter_add_(1, at, torch.full_like(lse, -1.0))
    g *= valid / count
    out["dh"], out["dw"], out["db"] = (g @ w32).to(h.dtype), (g.t() @ h32).to(w.dtype), g.sum(dim=0).to(b.dtype)
    return out


# ---- the framework's calls -------------------------------------------------------------------------------------------------
def _own(s):
    from pagraph_amd import ops
    case = s["case"]
    if case["op"] == "loss":
        if not case["train"]:                               # scoring: one loss a row
            return {"loss": ops.linear_cross_entropy(s["h"], s["lin"], s["labels"], reduction="none")}
        loss = ops.linear_cross_entropy(s["h"], s["lin"], s["labels"])
        dh, dw, db = torch.autograd.grad(loss, (s["h"], s["lin"].weight, s["lin"].bias))
        return {"loss": loss.detach(), "dh": dh, "dw": dw, "db": db}
    spec = ops.DropoutSpec(case["p"], s["key"][1], s["key"][2], s["step"]) if "key" in s else None
    if case["op"] == "dropout":
        y = ops.dropout(s["x"], spec)
        if not case["train"]:
            return {"y": y}
        return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["gy"])[0]}
    leaves = (s["x"], s["norm"].weight, s["norm"].bias)
    if "res" in s:
        y, total = ops.layer_norm(s["x"], s["norm"], residual=s["res"], dropout=spec)
        if not case["train"]:
            return {"s": total, "y": y}
        dx, dw, db, dres = torch.autograd.grad((y, total), leaves + (s["res"],), (s["gy"], s["gs"]))
        return {"s": total.detach(), "y": y.detach(), "dres": dres, "dx": dx, "dw": dw, "db": db}
    y = ops.layer_norm(s["x"], s["norm"])
    if not case["train"]:
        return {"y": y}
    dx, dw, db = torch.autograd.grad(y, leaves, s["gy"])
    return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}


def run(state):
    if own:
        return _own(state)
    return {"dropout": _plain_dropout, "norm": _plain_norm, "loss": _plain_loss}[state["case"]["op"]](state)


# ---- floors ----------------------------------------------------------------------------------------------------------------
def work(case):
    e, n, train = _BYTES[case["type"]], case["n"], case["train"]
    if case["op"] == "loss":
        k, c = case["k"], case["c"]
        read = (n * k + c * k + c) * e + 8 * n
        return {"bytes": read + ((n * k + c * k + c) * e + 4 if train else 4 * n), "flops": (6 if train else 2) * n * k * c}
    d = case["d"]
    if case["op"] == "dropout":
        return {"bytes": n * d * e * (4 if train else 2), "flops": n * d * (2 if train else 1)}
    passes = 4 if case["residual"] else 2                                    # x, y (residual, sum)
    if train:
        passes += 4 if case["residual"] else 2                               # gy, dx (the sum's gradient, the residual's)
    return {"bytes": n * d * e * passes + d * e * (4 if train else 2), "flops": n * d * (22 if train else 8)}


# ---- the operators' definitions in 64 bits ---------------------------------------------------------------------------------
def _mask64(n, d, key):
    """float64 [n, d]: 0 where dropped, the scale where kept, word by word from the mask's definition"""
    thr, seed, tag, step = key
    lo, sh = np.uint64(_M32), np.uint64(32)
    cols = np.arange(d)
    quads = np.unique((cols // 512) * 64 + (cols // 4) % 64)
    ctr = [np.broadcast_to(np.arange(n, dtype=np.uint64)[:, None], (n, len(quads))), np.broadcast_to(quads.astype(np.uint64), (n, len(quads))),
           np.full((n, len(quads)), tag, np.uint64), np.full((n, len(quads)), step, np.uint64)]
    ka, kb = seed & _M32, seed >> 32
    for _ in range(10):
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(b >> sh) ^ ctr[1] ^ np.uint64(ka), b & lo, (a >> sh) ^ ctr[3] ^ np.uint64(kb), a & lo]
        ka, kb = (ka + 0x9E3779B9) & _M32, (kb + 0xBB67AE85) & _M32
    out = np.empty((n, d))
    where = np.searchsorted(quads, (cols // 512) * 64 + (cols // 4) % 64)
    word = 2 * ((cols // 256) % 2) + (cols % 4) // 2
    for which in range(4):
        for odd in range(2):
            mine = (word == which) & (cols % 2 == odd)
            u = (ctr[which][:, where[mine]] >> np.uint64(16 * odd)) & np.uint64(0xFFFF)
            out[:, mine] = np.where(u >= np.uint64(thr), 65536.0 / (65536 - thr), 0.0)
    return torch.from_numpy(out)


def exact(case, seed):
    dev = torch.device("cuda")
    t = {name: v if v.dtype == torch.int64 else v.double() for name, v in _inputs(case, seed, dev).items()}
    key = _mask_key(case, seed)
    keep = _mask64(case["n"], case["d"], key).to(dev) if key is not None else 1.0
    if case["op"] == "dropout":
        return {"y": t["x"] * keep, **({"dx": t["gy"] * keep} if case["train"] else {})}
    if case["op"] == "norm":
        v = t["x"] * keep + t.get("res", 0.0)
        if "res" in t:
            # the rows handed on are held in the rows' type: that rounding is part of what is normalised
            v = v.float().to(_TYPES[case["type"]]).double()
        var, mean = torch.var_mean(v, dim=1, unbiased=False, keepdim=True)
        sd = (var + 1e-5).sqrt()
        unit = (v - mean) / sd
        out = {"s": v} if "res" in t else {}
        out["y"] = unit * t["w"] + t["b"]
        if case["train"]:
            up = t["gy"] * t["w"]
            back = (up - up.mean(1, True) - unit * (up * unit).mean(1, True)) / sd + t.get("gs", 0.0)
            if "res" in t:
                out["dres"] = back
            out.update(dx=back * keep, dw=(t["gy"] * unit).sum(0), db=t["gy"].sum(0))
        return out
    h, w, lab = t["h"], t["w"], t["labels"]
    seen = torch.nonzero((lab >= 0) & (lab < case["c"])).view(-1)
    each = torch.zeros(case["n"], dtype=torch.float64, device=dev)
    dh, dw, db = torch.zeros_like(h), torch.zeros_like(w), torch.zeros_like(t["b"])
    for rows in torch.split(seen, 2048):
        logp = torch.log_softmax(torch.addmm(t["b"], h[rows], w.t()), dim=1)
        here = torch.arange(rows.numel(), device=dev)
        each[rows] = -logp[here, lab[rows]]
        if case["train"]:
            p = logp.exp_()
            p[here, lab[rows]] -= 1.0
            p /= seen.numel()
            dh[rows] = p @ w
            dw += p.t() @ h[rows]
            db += p.sum(0)
    return {"loss": each.sum() / seen.numel(), "dh": dh, "dw": dw, "db": db} if case["train"] else {"loss": each}
