"""Operators of language models that stand beside the state-space operators, as a program calls them.

Four of them: the gated delta rule over whole sequences (a linear recurrence whose state is corrected by what it already holds, the
layer that models mix with state-space layers) and its single-token form, the log probabilities of given tokens with entropy and
top alternatives, and distillation from a teacher's top logits.  ``listed()`` names passes over the range of sizes, directions and
types, ``draw()`` gives more of the same ranges, ``prepare()`` makes what a program has in hand, ``run()`` makes one pass: with ``own``
through ``ssm_b200.ops``, otherwise in elementary torch operations in 32 bits.  ``exact()`` states the same in 64 bits from the
definitions (the recurrence token by token), ``work()`` the bytes and operations that a pass cannot do without.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
IGNORE = -100


def listed():
    return [
        # one long prompt: few heads, a long chain; keys shared by two value heads each
        {"name": "delta_prefill_long", "kind": "delta", "batch": 1, "len": 16384, "heads": 32, "key_heads": 16, "kdim": 128, "vdim": 128, "dtype": "bf16"},
        # a batch of prompts that fills the GPU
        {"name": "delta_prefill_batch", "kind": "delta", "batch": 8, "len": 4096, "heads": 16, "key_heads": 16, "kdim": 128, "vdim": 128, "dtype": "bf16"},
        # prompts of different lengths end to end, at the head sizes of this package's Mamba-2 layers (64 channels, 128 states)
        {"name": "delta_prefill_packed", "kind": "delta_packed", "sequences": 24, "len": 16384, "heads": 32, "key_heads": 32, "kdim": 128, "vdim": 64, "dtype": "f16"},
        # training: forward and backward; then a small one in full precision, of odd length and odd heads
        {"name": "delta_train", "kind": "delta_train", "batch": 2, "len": 4096, "heads": 16, "key_heads": 16, "kdim": 128, "vdim": 128, "dtype": "bf16"},
        {"name": "delta_train_f32", "kind": "delta_train", "batch": 1, "len": 777, "heads": 6, "key_heads": 3, "kdim": 64, "vdim": 96, "dtype": "f32"},
        # decoding: one user, then a served batch
        {"name": "delta_step_one", "kind": "delta_step", "batch": 1, "heads": 32, "key_heads": 16, "kdim": 128, "vdim": 128, "dtype": "bf16"},
        {"name": "delta_step_batch", "kind": "delta_step", "batch": 256, "heads": 32, "key_heads": 16, "kdim": 128, "vdim": 128, "dtype": "bf16"},
        # the answers of a decode step with their alternatives; scoring of a prompt; the policy term and entropy bonus of a training step
        {"name": "logp_decode_top", "kind": "logp", "rows": 8, "vocab": 50280, "top": 20, "dtype": "bf16"},
        {"name": "logp_score_prompt", "kind": "logp", "rows": 4096, "vocab": 50280, "top": 5, "dtype": "bf16"},
        {"name": "logp_train", "kind": "logp_train", "rows": 8192, "vocab": 50280, "dtype": "bf16"},
        # distillation steps: a few rows in full precision with an unpadded vocabulary, and a training batch
        {"name": "distill_small_f32", "kind": "distill", "rows": 60, "vocab": 50277, "top": 32, "dtype": "f32"},
        {"name": "distill_train", "kind": "distill", "rows": 4096, "vocab": 50280, "top": 64, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["delta", "delta", "delta_packed", "delta_train", "delta_train", "delta_step", "delta_step", "logp", "logp_train", "distill"])
    half = rng.choice(["bf16", "bf16", "f16"])
    anyt = rng.choice(["bf16", "f16", "f32"])
    if kind.startswith("delta"):
        if kind == "delta_step":
            c = {"batch": _log_int(rng, 1, 256)}
            dtype = anyt
        elif kind == "delta_packed":
            length = _log_int(rng, 64, 16384)
            c = {"sequences": _log_int(rng, 1, min(48, length)), "len": length}
            dtype = half
        else:
            length = _log_int(rng, 1, 16384 if kind == "delta" else 4096)
            c = {"batch": _log_int(rng, 1, 8), "len": length}
            dtype = half if kind == "delta" else rng.choice(["bf16", "bf16", "f16", "f32"])
        share = rng.choice([1, 1, 2, 4])
        most = {"delta": 524288, "delta_packed": 524288, "delta_train": 131072, "delta_step": 8192}[kind]
        if dtype == "f32" and kind == "delta_train":
            most = 16384
        tokens = c.get("batch", 1) * c.get("len", 1)
        heads = max(1, min(64, most // tokens // share)) if kind != "delta_step" else min(48, 8192 // tokens)
        heads = share * max(1, _log_int(rng, 1, max(1, heads // share)))
        if "batch" in c:
            while c["batch"] > 1 and c["batch"] * c.get("len", 1) * heads > most:
                c["batch"] -= 1
        if dtype == "f32":
            kd, vd = rng.choice([32, 64, 80, 128]), rng.choice([48, 64, 96, 128])
        else:
            kd, vd = rng.choice([64, 128, 128]), rng.choice([64, 128, 128])
        return {"kind": kind, **c, "heads": heads, "key_heads": heads // share, "kdim": kd, "vdim": vd, "dtype": dtype}
    vocab = _log_int(rng, 1000, 151936)
    if kind == "logp":
        return {"kind": kind, "rows": _log_int(rng, 1, max(1, 4096 * 50280 // vocab)), "vocab": vocab, "top": rng.choice([0, 1, 5, 20]), "dtype": anyt}
    if kind == "logp_train":
        return {"kind": kind, "rows": _log_int(rng, 16, max(16, 4096 * 50280 // vocab)), "vocab": vocab, "dtype": anyt}
    return {"kind": kind, "rows": _log_int(rng, 4, max(4, 2048 * 50280 // vocab)), "vocab": vocab, "top": rng.choice([8, 20, 50, 64]), "dtype": anyt}


# ---- inputs ------------------------------------------------------------------------------------------------------------------


def _delta_inputs(case, gen, lead):
    """What a layer hands to the operator for tokens of shape `lead`: keys and queries of norm one, log decays of the size that step
    sizes between 0.001 and 0.1 and rates between 1 and 16 give, write strengths from a sigmoid."""
    dt, dev = DTYPES[case["dtype"]], "cuda"
    h, hk, kd, vd = case["heads"], case["key_heads"], case["kdim"], case["vdim"]

    def unit(*shape):
        t = torch.randn(*shape, device=dev, generator=gen)
        return (t / t.norm(dim=-1, keepdim=True)).to(dt)

    rate = 1 + 15 * torch.rand(h, device=dev, generator=gen)
    step = torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(h, device=dev, generator=gen))
    bias = step + torch.log(-torch.expm1(-step))
    raw = torch.randn(*lead, h, device=dev, generator=gen) + bias
    g = -rate * torch.where(raw > 20, raw, torch.log1p(torch.exp(raw)))
    return {"q": unit(*lead, hk, kd), "k": unit(*lead, hk, kd), "v": torch.randn(*lead, h, vd, device=dev, generator=gen).to(dt), "g": g,
            "beta": torch.sigmoid(torch.randn(*lead, h, device=dev, generator=gen)).to(dt)}


def _cuts(case, gen):
    """Boundaries of packed sequences: uneven, all tokens covered."""
    n, length = case["sequences"], case["len"]
    w = torch.rand(n, generator=gen, device="cuda").cpu() + 0.05
    ends = torch.round(torch.cumsum(w, 0) / w.sum() * length).to(torch.int64)
    ends[-1] = length
    return torch.cat([torch.zeros(1, dtype=torch.int64), ends])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, dt = case["kind"], DTYPES[case["dtype"]]
    s = {"case": case, "kind": kind}
    if kind.startswith("delta"):
        lead = {"delta_step": (case.get("batch"),), "delta_packed": (1, case.get("len"))}.get(kind, (case.get("batch"), case.get("len")))
        s.update(_delta_inputs(case, gen, lead))
        shape = (case["heads"], case["vdim"], case["kdim"])
        if kind == "delta_step":
            s["state"] = 0.3 * torch.randn(case["batch"], *shape, device="cuda", generator=gen)
        elif kind == "delta_packed":
            cuts = _cuts(case, gen)
            s["cu"], s["longest"] = cuts.cuda(), int((cuts[1:] - cuts[:-1]).max())
        elif kind == "delta_train":
            s["g"] = s["g"].to(dt)  # the training step keeps its activations in one type
            s["do"] = torch.randn(*s["v"].shape, device="cuda", generator=gen).to(dt)
            for n in ("q", "k", "v", "g", "beta"):
                s[n].requires_grad_(True)
        return s
    rows, vocab = case["rows"], case["vocab"]
    logits = 2.5 * torch.randn(rows, vocab, device="cuda", generator=gen)
    targets = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    logits.scatter_add_(1, targets[:, None], 8 * torch.rand(rows, 1, device="cuda", generator=gen))
    s["targets"] = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.1, torch.full_like(targets, IGNORE), targets)
    if kind == "distill":
        noisy = logits + torch.randn(rows, vocab, device="cuda", generator=gen)
        top, ids = torch.topk(noisy, case["top"], dim=-1)
        s["teacher"], s["ids"] = top.to(dt), ids
        del noisy
    s["logits"] = logits.to(dt)
    loss_scale = 4096.0 if case["dtype"] == "f16" else 1.0 / rows  # fp16 training scales its loss so that small gradients keep their bits
    s["w"] = torch.randn(rows, device="cuda", generator=gen) * loss_scale
    s["wh"] = 0.01 * torch.randn(rows, device="cuda", generator=gen) * loss_scale
    if kind in ("logp_train", "distill"):
        s["logits"].requires_grad_(True)
    return s


# ---- plain forms in 32 bits --------------------------------------------------------------------------------------------------

CHUNK = 64


def _plain_chunks(q, k, v, g, beta, scale):
    """The gated delta rule on (B, L, H, .) in 32 bits, cut into chunks: within one, the corrected values of all tokens solve a unit
    lower triangular system, whose inverse is a product of powers; from one to the next the state (B, H, K, V) is carried."""
    nb, nl, nh, kd = k.shape
    vd, n = v.shape[-1], -(-nl // CHUNK)

    def cut(t):  # (B, L, H, ...) -> (B, H, n, CHUNK, ...); tokens behind the end change nothing (no key, no strength, no decay)
        t = torch.cat([t, t.new_zeros(nb, n * CHUNK - nl, *t.shape[2:])], 1)
        return t.reshape(nb, n, CHUNK, *t.shape[2:]).transpose(2, 3).transpose(1, 2)

    q, k, v, g, beta = cut(q * scale), cut(k), cut(v), cut(g), cut(beta)
    c = torch.cumsum(g.double(), -1)
    row = torch.arange(CHUNK, device=q.device)
    low, strict = row[:, None] >= row[None, :], row[:, None] > row[None, :]
    decay = torch.exp(torch.where(low, c[..., :, None] - c[..., None, :], torch.full((), -math.inf, dtype=c.dtype, device=c.device))).float()
    into, out_of, whole = torch.exp(c).float(), torch.exp(c[..., -1:] - c).float(), torch.exp(c[..., -1]).float()
    power = torch.where(strict, -beta[..., :, None] * decay * (k @ k.transpose(-1, -2)), torch.zeros((), device=q.device))
    inverse = torch.eye(CHUNK, device=q.device) + power
    for _ in range(5):
        power = power @ power
        inverse = inverse + inverse @ power
    mixed = decay * (q @ k.transpose(-1, -2))
    state, outs = q.new_zeros(nb, nh, kd, vd), []
    for i in range(n):
        rest = v[:, :, i] - into[:, :, i, :, None] * (k[:, :, i] @ state)
        u = inverse[:, :, i] @ (beta[:, :, i, :, None] * rest)
        outs.append(into[:, :, i, :, None] * (q[:, :, i] @ state) + mixed[:, :, i] @ u)
        state = whole[:, :, i, None, None] * state + (out_of[:, :, i, :, None] * k[:, :, i]).transpose(-1, -2) @ u
    o = torch.stack(outs, 2).transpose(1, 2).transpose(2, 3).reshape(nb, n * CHUNK, nh, vd)
    return o[:, :nl], state.transpose(-1, -2)


def _plain_delta(q, k, v, g, beta, scale):
    rep = v.shape[2] // k.shape[2]
    q, k = (t.float().repeat_interleave(rep, 2) for t in (q, k))
    return _plain_chunks(q, k, v.float(), g.float(), beta.float(), scale)


def _rows_of(s):
    """Packed tokens as a padded batch: for every sequence and step the token's place, and whether there is one."""
    start, end = s["cu"][:-1], s["cu"][1:]
    at = start[:, None] + torch.arange(s["longest"], device=start.device)
    live = at < end[:, None]
    return torch.where(live, at, torch.zeros_like(at)), live


def _run_plain(s):
    kind, case = s["kind"], s["case"]
    if kind.startswith("delta"):
        scale = case["kdim"] ** -0.5
        names = ("q", "k", "v", "g", "beta")
        if kind == "delta":
            o, state = _plain_delta(*(s[n] for n in names), scale)
            return {"o": o.to(s["v"].dtype), "state": state.to(s["v"].dtype)}
        if kind == "delta_packed":
            at, live = _rows_of(s)
            padded = []
            for n in names:
                t = s[n][0][at].float()
                padded.append(t * live.reshape(*live.shape, *(1,) * (t.dim() - 2)))
            o, state = _plain_delta(*padded, scale)
            out = torch.zeros(s["v"].shape[1:], device=o.device)
            out[at[live]] = o[live]
            return {"o": out[None].to(s["v"].dtype), "state": state.to(s["v"].dtype)}
        if kind == "delta_train":
            leaves = [s[n] for n in names]
            o, _ = _plain_delta(*leaves, scale)
            o = o.to(s["v"].dtype)
            return {"o": o.detach(), **dict(zip(("dq", "dk", "dv", "dg", "dbeta"), torch.autograd.grad(o, leaves, s["do"])))}
        q, k, v, g, beta = (s[n].float() for n in names)
        rep = case["heads"] // case["key_heads"]
        q, k = q.repeat_interleave(rep, 1) * scale, k.repeat_interleave(rep, 1)
        state = s["state"] * torch.exp(g)[..., None, None]
        u = beta[..., None] * (v - (state * k[:, :, None]).sum(-1))
        state = state + u[..., None] * k[:, :, None]
        s["state"].copy_(state)
        return {"o": (state * q[:, :, None]).sum(-1).to(s["v"].dtype), "state": s["state"]}
    x = s["logits"].float()
    if kind == "distill":
        tau = 2.0
        x = x / tau
        t = s["teacher"].float() / tau
        logt = t - t.amax(-1, keepdim=True)
        logt = logt - torch.log(torch.exp(logt).sum(-1, keepdim=True))
        m = x.detach().amax(-1, keepdim=True)
        logz = torch.log(torch.exp(x - m).sum(-1, keepdim=True)) + m
        loss = (torch.exp(logt) * (logt - (torch.gather(x, 1, s["ids"]) - logz))).sum(-1)
        return {"loss": loss.detach(), "dlogits": torch.autograd.grad(loss, s["logits"], s["w"])[0]}
    m = x.detach().amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    logz = torch.log(z) + m
    kept = s["targets"] != IGNORE
    logp = torch.where(kept, (torch.gather(x, 1, torch.where(kept, s["targets"], torch.zeros_like(s["targets"]))[:, None]) - logz)[:, 0], torch.zeros((), device=x.device))
    entropy = torch.log(z)[:, 0] - (e * (x - m)).sum(-1) / z[:, 0]
    if kind == "logp_train":
        got = torch.autograd.grad([logp, entropy], s["logits"], [s["w"], s["wh"]])[0]
        return {"logp": logp.detach(), "entropy": entropy.detach(), "dlogits": got}
    out = {"logp": logp, "entropy": entropy}
    if case["top"]:
        top, ids = torch.sort(x, dim=-1, descending=True, stable=True)
        out["top"], out["ids"] = (top[:, :case["top"]] - logz), ids[:, :case["top"]].clone()
    return out


# ---- the framework's calls ---------------------------------------------------------------------------------------------------


def _run_own(s):
    from ssm_b200 import ops

    kind, case = s["kind"], s["case"]
    if kind == "delta":
        o, state = ops.gated_delta_scan(s["q"], s["k"], s["v"], s["g"], s["beta"], return_final_state=True)
        return {"o": o, "state": state}
    if kind == "delta_packed":
        o, state = ops.gated_delta_scan(s["q"], s["k"], s["v"], s["g"], s["beta"], cu_seqlens=s["cu"], return_final_state=True)
        return {"o": o, "state": state}
    if kind == "delta_train":
        leaves = [s[n] for n in ("q", "k", "v", "g", "beta")]
        o = ops.gated_delta_scan(*leaves)
        return {"o": o.detach(), **dict(zip(("dq", "dk", "dv", "dg", "dbeta"), torch.autograd.grad(o, leaves, s["do"])))}
    if kind == "delta_step":
        return {"o": ops.gated_delta_step(s["state"], s["q"], s["k"], s["v"], s["g"], s["beta"]), "state": s["state"]}
    if kind == "distill":
        loss = ops.topk_distill_loss(s["logits"], s["teacher"], s["ids"], temperature=2.0)
        return {"loss": loss.detach(), "dlogits": torch.autograd.grad(loss, s["logits"], s["w"])[0]}
    if kind == "logp_train":
        logp, entropy = ops.token_log_probs(s["logits"], s["targets"], return_entropy=True)
        got = torch.autograd.grad([logp, entropy], s["logits"], [s["w"], s["wh"]])[0]
        return {"logp": logp.detach(), "entropy": entropy.detach(), "dlogits": got}
    if not case["top"]:
        logp, entropy = ops.token_log_probs(s["logits"], s["targets"], return_entropy=True)
        return {"logp": logp, "entropy": entropy}
    logp, entropy, top, ids = ops.token_log_probs(s["logits"], s["targets"], return_entropy=True, top_k=case["top"])
    return {"logp": logp, "entropy": entropy, "top": top, "ids": ids}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------


def _exact_scan(q, k, v, g, beta, scale, do=None):
    """Token by token on (B, L, H, .) doubles: S' = exp(g) S, r = v - S'^T k, S = S' + beta k r^T, o = scale S^T q, the state S held as
    (K, V); and the same walked back for the gradients."""
    nb, nl, nh, kd = k.shape
    vd = v.shape[-1]
    first = lambda t: t.transpose(0, 1).contiguous()  # noqa: E731
    q, k, v, a, beta = first(q), first(k), first(v), first(torch.exp(g)), first(beta)
    state = torch.zeros(nb, nh, kd, vd, dtype=torch.float64, device=q.device)
    o, rest, states = torch.empty_like(v), torch.empty_like(v), [state]
    for t in range(nl):
        old = a[t][..., None, None] * state
        r = v[t] - (k[t][..., None, :] @ old)[..., 0, :]
        state = old + (beta[t][..., None] * k[t])[..., None] * r[..., None, :]
        o[t] = scale * (q[t][..., None, :] @ state)[..., 0, :]
        if do is not None:
            rest[t] = r
            states.append(state)
    back = lambda t: t.transpose(0, 1)  # noqa: E731
    if do is None:
        return back(o), state.transpose(-1, -2)
    do = first(do)
    ds = torch.zeros_like(state)
    dq, dk, dv, dg, db = (torch.empty_like(t) for t in (q, k, v, a, beta))
    for t in range(nl - 1, -1, -1):
        dq[t] = scale * (states[t + 1] @ do[t][..., None])[..., 0]
        ds = ds + scale * q[t][..., None] * do[t][..., None, :]
        y = (ds @ rest[t][..., None])[..., 0]
        db[t] = (y * k[t]).sum(-1)
        w = beta[t][..., None] * (k[t][..., None, :] @ ds)[..., 0, :]
        dv[t] = w
        old = a[t][..., None, None] * states[t]
        dk[t] = beta[t][..., None] * y - (old @ w[..., None])[..., 0]
        ds = ds - k[t][..., None] * w[..., None, :]
        dg[t] = (ds * old).sum((-1, -2))
        ds = a[t][..., None, None] * ds
    return back(o), [back(x) for x in (dq, dk, dv, dg, db)]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind.startswith("delta"):
            rep, scale = case["heads"] // case["key_heads"], case["kdim"] ** -0.5
            q, k, v, g, beta = (s[n].double() for n in ("q", "k", "v", "g", "beta"))
            head = 1 if kind == "delta_step" else 2
            q, k = q.repeat_interleave(rep, head), k.repeat_interleave(rep, head)
            if kind == "delta_step":
                state = s["state"].double() * torch.exp(g)[..., None, None]
                rest = v - torch.einsum("bhvk,bhk->bhv", state, k)
                state = state + torch.einsum("bhv,bhk->bhvk", beta[..., None] * rest, k)
                return {"o": scale * torch.einsum("bhvk,bhk->bhv", state, q), "state": state}
            if kind == "delta":
                o, state = _exact_scan(q, k, v, g, beta, scale)
                return {"o": o, "state": state}
            if kind == "delta_packed":
                cu = s["cu"].tolist()
                outs, states = [], []
                if case["len"] > 20000:
                    return None
                for a, b in zip(cu, cu[1:]):
                    o, state = _exact_scan(*(t[:, a:b] for t in (q, k, v, g, beta)), scale)
                    outs.append(o)
                    states.append(state)
                return {"o": torch.cat(outs, 1), "state": torch.cat(states)}
            o, (dq, dk, dv, dg, db) = _exact_scan(q, k, v, g, beta, scale, s["do"].double())
            fold = lambda t: t.reshape(*t.shape[:2], case["key_heads"], rep, t.shape[-1]).sum(3)  # noqa: E731
            return {"o": o, "dq": fold(dq), "dk": fold(dk), "dv": dv, "dg": dg, "dbeta": db}
        x = s["logits"].detach().double()
        if kind == "distill":
            logq = torch.log_softmax(x / 2.0, -1)
            logt = torch.log_softmax(s["teacher"].double() / 2.0, -1)
            pt = torch.exp(logt)
            loss = (pt * (logt - torch.gather(logq, 1, s["ids"]))).sum(-1)
            d = torch.exp(logq).scatter_add_(1, s["ids"], -pt) * (s["w"].double()[:, None] / 2.0)
            return {"loss": loss, "dlogits": d}
        logp_all = torch.log_softmax(x, -1)
        kept = s["targets"] != IGNORE
        at = torch.where(kept, s["targets"], torch.zeros_like(s["targets"]))[:, None]
        logp = torch.where(kept, torch.gather(logp_all, 1, at)[:, 0], torch.zeros((), dtype=torch.float64, device=x.device))
        p = torch.exp(logp_all)
        entropy = -(p * logp_all).sum(-1)
        if kind == "logp_train":
            wl = torch.where(kept, s["w"].double(), torch.zeros((), dtype=torch.float64, device=x.device))
            d = -p * (wl[:, None] + s["wh"].double()[:, None] * (logp_all + entropy[:, None]))
            d.scatter_add_(1, at, wl[:, None])
            return {"logp": logp, "entropy": entropy, "dlogits": d}
        if not case["top"]:
            return {"logp": logp, "entropy": entropy}
        top, ids = torch.sort(logp_all, dim=-1, descending=True, stable=True)
        return {"logp": logp, "entropy": entropy, "top": top[:, :case["top"]], "ids": None}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------


def work(case):
    kind, size = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind.startswith("delta"):
        h, hk, kd, vd = case["heads"], case["key_heads"], case["kdim"], case["vdim"]
        tokens = case.get("batch", 1) * case.get("len", 1)
        states = h * kd * vd * case.get("sequences", case.get("batch", 1))
        qk, vo = 2 * hk * kd * size, h * vd * size
        gb = h * (4 + size)
        once = 6 * h * kd * vd  # a token's products with the state: what it holds for the key, the correction, the answer
        if kind == "delta_step":
            return {"bytes": tokens * (qk + 2 * vo + gb) + 2 * 4 * states, "flops": tokens * once}
        if kind == "delta_train":  # reads q, k, v, g, beta, do; writes o and five gradients; forward once, twice that back
            gb = h * 2 * size
            return {"bytes": tokens * (2 * qk + 4 * vo + 2 * gb), "flops": 3 * tokens * once}
        return {"bytes": tokens * (qk + 2 * vo + gb) + size * states, "flops": tokens * once}
    rows, vocab = case["rows"], case["vocab"]
    if kind == "logp":
        return {"bytes": rows * (vocab * size + 8 + 8 + 12 * case["top"]), "flops": 5 * rows * vocab}
    if kind == "logp_train":
        return {"bytes": rows * (2 * vocab * size + 8 + 8 + 8), "flops": 10 * rows * vocab}
    return {"bytes": rows * (2 * vocab * size + case["top"] * (8 + size) + 8), "flops": 8 * rows * vocab}
