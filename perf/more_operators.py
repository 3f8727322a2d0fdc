"""What a training step of a language model runs around its mixers, as a program calls it.

Three operators: the norms after and before a block fused with the block's gate, its residual scale and the residual add (``fused_block_norm``),
softmax cross entropy straight from hidden states and the head's weight, without keeping the logits (``linear_cross_entropy``), and the
norm over all gradients with clipping (``global_norm``, ``clip_global_norm_``).  ``listed()`` names passes over the range of sizes,
directions and types, ``draw()`` gives more of the same ranges, ``prepare()`` makes what a program has in hand, ``run()`` makes one
pass: with ``own`` through ``ssm_b200.ops``, otherwise in elementary torch operations in 32 bits.  ``exact()`` states the same in 64 bits
from the definitions, ``work()`` the bytes and operations that a pass cannot do without.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
IGNORE = -100
EPS = 1e-5


def listed():
    return [
        # a decode step of a served batch: one token a sequence, the residual stream in 32 bits, a learned gate per channel
        {"name": "norm_decode", "kind": "norm", "batch": 8, "len": 1, "dim": 2560, "gate": "channel", "rms": True, "dtype": "bf16"},
        # one long prompt, no gate
        {"name": "norm_prefill", "kind": "norm", "batch": 1, "len": 32768, "dim": 2560, "gate": "none", "rms": True, "dtype": "bf16"},
        # training: forward and backward, the gate given per sequence; then a small one in full precision, LayerNorm of odd width, a gate per token
        {"name": "norm_train", "kind": "norm_train", "batch": 4, "len": 4096, "dim": 2560, "gate": "sequence", "rms": True, "dtype": "bf16"},
        {"name": "norm_train_f32", "kind": "norm_train", "batch": 3, "len": 777, "dim": 1001, "gate": "token", "rms": False, "dtype": "f32"},
        # the loss of a few tokens; of a batch of evaluation
        {"name": "loss_few", "kind": "loss", "rows": 7, "dim": 768, "vocab": 50277, "dtype": "bf16"},
        {"name": "loss_eval", "kind": "loss", "rows": 4096, "dim": 2560, "vocab": 50280, "dtype": "bf16"},
        # training steps: the mean over a batch; an odd number of tokens and an unpadded vocabulary with a scaled loss; per-token weights and a
        # penalty on log Z in full precision
        {"name": "loss_train", "kind": "loss_train", "rows": 8192, "dim": 2560, "vocab": 50280, "reduction": "mean", "dtype": "bf16"},
        {"name": "loss_train_odd", "kind": "loss_train", "rows": 1999, "dim": 1024, "vocab": 50277, "reduction": "mean", "dtype": "f16"},
        {"name": "loss_train_f32", "kind": "loss_train", "rows": 500, "dim": 512, "vocab": 16003, "reduction": "none", "dtype": "f32"},
        # gradients of whole models: the norm alone of a small one (many small tensors), clipping of a small and of a large one
        {"name": "grads_norm_small", "kind": "grads_norm", "layers": 24, "dim": 160, "vocab": 5003, "dtype": "f32"},
        {"name": "grads_clip_small", "kind": "grads_clip", "layers": 24, "dim": 768, "vocab": 50280, "dtype": "bf16"},
        {"name": "grads_clip_large", "kind": "grads_clip", "layers": 64, "dim": 2560, "vocab": 50280, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm_train", "norm_train", "loss", "loss_train", "loss_train", "loss_train", "grads_norm", "grads_clip", "grads_clip"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind.startswith("norm"):
        dim = _log_int(rng, 64, 5120)
        if rng.random() < 0.6:
            dim = max(64, dim // 64 * 64)
        most = (32768 if kind == "norm" else 16384) * 2560 // dim
        batch = _log_int(rng, 1, min(64, most))
        length = _log_int(rng, 1, max(1, min(32768, most // batch)))
        return {"kind": kind, "batch": batch, "len": length, "dim": dim, "gate": rng.choice(["none", "channel", "sequence", "token"]), "rms": rng.random() < 0.7,
                "dtype": dtype}
    if kind.startswith("loss"):
        dim = _log_int(rng, 64, 2560)
        if rng.random() < 0.6:
            dim = max(64, dim // 64 * 64)
        vocab = _log_int(rng, 500, 151936)
        most = (4096 if kind == "loss" else 8192) * 50280 * 2560 // (vocab * dim)
        if dtype == "f32":
            most //= 4
        rows = _log_int(rng, 1, max(1, min(16384, most, 2 ** 30 // vocab)))
        c = {"kind": kind, "rows": rows, "dim": dim, "vocab": vocab, "dtype": dtype}
        if kind == "loss_train":
            c["reduction"] = rng.choice(["mean", "mean", "sum", "none"])
        return c
    dim = _log_int(rng, 8, 320) * 8
    layers = _log_int(rng, 1, 64)
    vocab = _log_int(rng, 500, 50280)
    if dtype == "f32":
        layers = min(layers, 32)
    return {"kind": kind, "layers": layers, "dim": dim, "vocab": vocab, "dtype": dtype}


# ---- inputs ------------------------------------------------------------------------------------------------------------------


def _shapes(case):
    """Parameters of a stack of state-space layers with a tied embedding: (shape, whether it is held in 32 bits whatever the model's type)."""
    d, heads, n = case["dim"], max(1, case["dim"] // 32), 128
    di = 2 * d
    layer = [((d,), False), ((di, d), False), ((di, d), False), ((n, d), False), ((n, d), False), ((heads, d), False), ((di, 4), False), ((n, 4), False),
             ((n, 4), False), ((di,), False), ((n,), False), ((n,), False), ((heads,), True), ((heads,), True), ((heads,), True), ((di,), False), ((d, di), False)]
    return [((case["vocab"], d), False)] + layer * case["layers"] + [((d,), False)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    s = {"case": case, "kind": kind}

    def rn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if kind.startswith("norm"):
        nb, nl, d = case["batch"], case["len"], case["dim"]
        s["x"] = (0.3 * rn(nb, nl, d)).to(dt)
        s["residual"] = 2 * rn(nb, nl, d)  # the stream is kept in 32 bits
        s["post_weight"], s["weight"] = (1 + 0.1 * rn(d)).to(dt), (1 + 0.1 * rn(d)).to(dt)
        s["post_bias"], s["bias"] = (None, None) if case["rms"] else ((0.1 * rn(d)).to(dt), (0.1 * rn(d)).to(dt))
        shape = {"none": None, "channel": (d,), "sequence": (nb, d), "token": (nb, nl, d)}[case["gate"]]
        s["gate"] = None if shape is None else (0.5 + 0.2 * rn(*shape)).to(dt)
        s["scale"] = 0.7
        if kind == "norm_train":
            s["dy"], s["dr"] = rn(nb, nl, d).to(dt), rn(nb, nl, d)
            for n in _norm_leaves(s):
                s[n].requires_grad_(True)
        return s
    if kind.startswith("loss"):
        rows, d, vocab = case["rows"], case["dim"], case["vocab"]
        weight = 2.5 / math.sqrt(d) * rn(vocab, d)
        targets = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
        raised = weight[targets]
        hidden = rn(rows, d) + 8 * torch.rand(rows, 1, device="cuda", generator=gen) * raised / (raised * raised).sum(-1, keepdim=True)
        s["hidden"], s["weight"] = hidden.to(dt), weight.to(dt)
        s["targets"] = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.1, torch.full_like(targets, IGNORE), targets)
        if kind == "loss_train":
            scale = 4096.0 if case["dtype"] == "f16" else 1.0  # fp16 training scales its loss so that small gradients keep their bits
            if case["reduction"] == "none":
                s["w"], s["wz"] = torch.rand(rows, device="cuda", generator=gen) * scale / rows, 1e-2 * rn(rows) * scale / rows
            else:
                s["w"] = torch.full((), scale if case["reduction"] == "mean" else scale / rows, device="cuda")
            s["hidden"].requires_grad_(True), s["weight"].requires_grad_(True)
        return s
    # one buffer a type, as a trainer keeps its gradients; each tensor on a 256-byte boundary, as a tensor of its own would be
    places, ends = [], {}
    for shape, wide in _shapes(case):
        t = torch.float32 if wide else dt
        at = ends.get(t, 0)
        places.append((shape, t, at))
        ends[t] = at + -(-math.prod(shape) // 128) * 128
    s["flat"] = {t: torch.zeros(n, dtype=t, device="cuda") for t, n in ends.items()}
    s["grads"] = [s["flat"][t][at:at + math.prod(shape)].view(shape) for shape, t, at in places]
    for g in s["grads"]:
        size = 10 ** (1 - 4 * torch.rand(1, device="cuda", generator=gen)) / math.sqrt(g.shape[-1])
        g.copy_(size * rn(*g.shape))
    s["limit"] = 1.0
    return s


def _norm_leaves(s):
    return [n for n in ("x", "residual", "post_weight", "weight", "post_bias", "bias", "gate") if s[n] is not None]


# ---- plain forms in 32 bits --------------------------------------------------------------------------------------------------


def _norm_rows(x, weight, bias, rms, eps):
    if not rms:
        x = x - x.mean(-1, keepdim=True)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight
    return x if bias is None else x + bias


def _block_norm(s, cast):
    """The definition on operands cast by `cast`: (y, new residual)."""
    x, residual, pw, w = (cast(s[n]) for n in ("x", "residual", "post_weight", "weight"))
    pb, b, gate = (None if s[n] is None else cast(s[n]) for n in ("post_bias", "bias", "gate"))
    rms = s["case"]["rms"]
    n = _norm_rows(x, pw, pb, rms, EPS)
    if gate is not None:
        n = n * (gate[:, None] if gate.dim() == 2 else gate)
    r = residual + s["scale"] * n
    return _norm_rows(r, w, b, rms, EPS), r


def _run_plain(s):
    kind, case = s["kind"], s["case"]
    if kind == "norm":
        with torch.no_grad():
            y, r = _block_norm(s, torch.Tensor.float)
        return {"y": y.to(s["x"].dtype), "residual": r}
    if kind == "norm_train":
        names = _norm_leaves(s)
        y, r = _block_norm(s, torch.Tensor.float)
        y = y.to(s["x"].dtype)
        got = torch.autograd.grad([y, r], [s[n] for n in names], [s["dy"], s["dr"]])
        return {"y": y.detach(), "residual": r.detach(), **{"d" + n: g for n, g in zip(names, got)}}
    if kind.startswith("loss"):
        train = kind == "loss_train"
        with torch.set_grad_enabled(train):
            z = s["hidden"].float() @ s["weight"].float().t()
            m = z.detach().amax(-1, keepdim=True)
            log_z = (torch.log(torch.exp(z - m).sum(-1, keepdim=True)) + m)[:, 0]
            kept = s["targets"] != IGNORE
            at = torch.where(kept, s["targets"], torch.zeros_like(s["targets"]))
            loss = torch.where(kept, log_z - torch.gather(z, 1, at[:, None])[:, 0], torch.zeros((), device=z.device))
        if not train:
            return {"loss": loss}
        leaves = [s["hidden"], s["weight"]]
        if case["reduction"] == "none":
            log_z = torch.where(kept, log_z, torch.zeros((), device=z.device))
            dh, dw = torch.autograd.grad([loss, log_z], leaves, [s["w"], s["wz"]])
            return {"loss": loss.detach(), "log_z": log_z.detach(), "dhidden": dh, "dweight": dw}
        loss = loss.sum()
        if case["reduction"] == "mean":
            loss = loss / torch.clamp(kept.sum(), min=1)
        dh, dw = torch.autograd.grad(loss, leaves, s["w"])
        return {"loss": loss.detach(), "dhidden": dh, "dweight": dw}
    norm = torch.sqrt(torch.stack([(g.float() * g.float()).sum(dtype=torch.float64) for g in s["grads"]]).sum()).float()
    if kind == "grads_norm":
        return {"norm": norm}
    coef = torch.clamp(s["limit"] / (norm + 1e-6), max=1.0)
    s["limit"] *= 0.999
    for g in s["grads"]:
        g.copy_(g.float() * coef)
    return {"norm": norm, **{str(t): flat for t, flat in s["flat"].items()}}


# ---- the framework's calls ---------------------------------------------------------------------------------------------------


def _run_own(s):
    from ssm_b200 import ops

    kind, case = s["kind"], s["case"]
    if kind.startswith("norm"):
        y, r = ops.fused_block_norm(s["x"], s["residual"], s["post_weight"], s["weight"], post_bias=s["post_bias"], bias=s["bias"], gate=s["gate"],
                                    residual_scale=s["scale"], is_rms=case["rms"], eps=EPS, residual_in_fp32=True)
        if kind == "norm":
            return {"y": y, "residual": r}
        names = _norm_leaves(s)
        got = torch.autograd.grad([y, r], [s[n] for n in names], [s["dy"], s["dr"]])
        return {"y": y.detach(), "residual": r.detach(), **{"d" + n: g for n, g in zip(names, got)}}
    if kind == "loss":
        return {"loss": ops.linear_cross_entropy(s["hidden"], s["weight"], s["targets"])}
    if kind == "loss_train":
        leaves = [s["hidden"], s["weight"]]
        if case["reduction"] == "none":
            loss, log_z = ops.linear_cross_entropy(s["hidden"], s["weight"], s["targets"], return_log_z=True)
            dh, dw = torch.autograd.grad([loss, log_z], leaves, [s["w"], s["wz"]])
            return {"loss": loss.detach(), "log_z": log_z.detach(), "dhidden": dh, "dweight": dw}
        loss = ops.linear_cross_entropy(s["hidden"], s["weight"], s["targets"], reduction=case["reduction"])
        dh, dw = torch.autograd.grad(loss, leaves, s["w"])
        return {"loss": loss.detach(), "dhidden": dh, "dweight": dw}
    if kind == "grads_norm":
        return {"norm": ops.global_norm(s["grads"])}
    norm = ops.clip_global_norm_(s["grads"], s["limit"])
    s["limit"] *= 0.999  # a limit that falls from step to step, so that every step clips
    return {"norm": norm, **{str(t): flat for t, flat in s["flat"].items()}}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------


def _exact_norm_back(x, weight, rms, eps, dy):
    """Gradient of weight * (x - mean) / std (mean 0 where `rms`): with h the normed row and g = weight dy, (g - [mean g] - h mean(g h)) / std."""
    c = x if rms else x - x.mean(-1, keepdim=True)
    inv = (c.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    h, g = c * inv, dy * weight
    d = g - h * (g * h).mean(-1, keepdim=True)
    if not rms:
        d = d - g.mean(-1, keepdim=True)
    return d * inv, h


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind.startswith("norm"):
            y, r = _block_norm(s, torch.Tensor.double)
            out = {"y": y, "residual": r}
            if kind == "norm":
                return out
            rms, d = case["rms"], case["dim"]
            dy = s["dy"].double()
            dr, h = _exact_norm_back(r, s["weight"].double(), rms, EPS, dy)
            dr = dr + s["dr"].double()
            gate = None if s["gate"] is None else s["gate"].double()
            wide = None if gate is None else gate[:, None] if gate.dim() == 2 else gate
            dn = s["scale"] * dr * (1.0 if wide is None else wide)
            dx, hx = _exact_norm_back(s["x"].double(), s["post_weight"].double(), rms, EPS, dn)
            rows = lambda t: t.reshape(-1, d).sum(0)  # noqa: E731
            out.update(dx=dx, dresidual=dr, dpost_weight=rows(dn * hx), dweight=rows(dy * h))
            if not rms:
                out.update(dpost_bias=rows(dn), dbias=rows(dy))
            if gate is not None:
                n = hx * s["post_weight"].double()
                if s["post_bias"] is not None:
                    n = n + s["post_bias"].double()
                dg = s["scale"] * dr * n
                out["dgate"] = rows(dg) if gate.dim() == 1 else dg.sum(1) if gate.dim() == 2 else dg
            return out
        if kind.startswith("loss"):
            h, w, t = s["hidden"].detach().double(), s["weight"].detach().double(), s["targets"]
            kept = t != IGNORE
            train = kind == "loss_train"
            none = train and case["reduction"] == "none"
            loss, log_z = h.new_zeros(h.shape[0]), h.new_zeros(h.shape[0])
            if train:
                share = s["w"].double()
                if case["reduction"] == "mean":
                    share = share / max(1, int(kept.sum()))
                share = share * kept
                share_z = s["wz"].double() * kept if none else torch.zeros_like(share)
                dh, dw = torch.empty_like(h), torch.zeros_like(w)
            step = max(1, 2 ** 26 // w.shape[0])
            for a in range(0, h.shape[0], step):
                b = min(h.shape[0], a + step)
                z = h[a:b] @ w.t()
                logp = torch.log_softmax(z, -1)
                at = torch.where(kept[a:b], t[a:b], torch.zeros_like(t[a:b]))[:, None]
                loss[a:b] = -torch.gather(logp, 1, at)[:, 0] * kept[a:b]
                log_z[a:b] = torch.logsumexp(z, -1) * kept[a:b]
                if train:
                    g = torch.exp(logp) * (share + share_z)[a:b, None]
                    g.scatter_add_(1, at, -share[a:b, None])
                    dh[a:b] = g @ w
                    dw += g.t() @ h[a:b]
            if not train:
                return {"loss": loss}
            if none:
                return {"loss": loss, "log_z": log_z, "dhidden": dh, "dweight": dw}
            total = loss.sum()
            if case["reduction"] == "mean":
                total = total / max(1, int(kept.sum()))
            return {"loss": total, "dhidden": dh, "dweight": dw}
        total = 0.0
        for g in s["grads"]:
            total += float(torch.linalg.vector_norm(g.double())) ** 2
        norm = torch.tensor(math.sqrt(total), dtype=torch.float64, device="cuda")
        if kind == "grads_norm":
            return {"norm": norm}
        coef = min(1.0, s["limit"] / (float(norm) + 1e-6))
        return {"norm": norm, **{str(t): flat.double() * coef for t, flat in s["flat"].items()}}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------


def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind.startswith("norm"):
        nb, d = case["batch"], case["dim"]
        n = nb * case["len"] * d
        gate = {"none": 0, "channel": d, "sequence": nb * d, "token": n}[case["gate"]] * size
        params = (2 if case["rms"] else 4) * d * size
        if kind == "norm":  # reads x and the residual, writes y and the new one
            return {"bytes": n * (2 * size + 8) + gate + params, "flops": 10 * n}
        # and back: reads the two gradients, writes those of x and of the residual, of the gate and of the parameters
        return {"bytes": n * (4 * size + 16) + 2 * gate + 2 * params, "flops": 35 * n}
    if kind.startswith("loss"):
        rows, d, vocab = case["rows"], case["dim"], case["vocab"]
        operands = (rows + vocab) * d * size + rows * 8
        if kind == "loss":
            return {"bytes": operands + 4 * rows, "flops": 2 * rows * d * vocab}
        return {"bytes": 2 * operands + 4 * rows, "flops": 6 * rows * d * vocab}
    total = held = 0
    for shape, wide in _shapes(case):
        n = math.prod(shape)
        total += n
        held += n * (4 if wide else size)
    if kind == "grads_norm":
        return {"bytes": held + 4, "flops": 2 * total}
    return {"bytes": 2 * held + 4, "flops": 3 * total}
