"""Cases and plain forms of three operators: cross attention to an encoder's states of another length, rotary positions with
several axes, and distillation from a teacher's top logits.

`run` computes them in elementary torch operations (32 bits, angles and remainders of probabilities in 64) or, where `own` is true, through
`lightly_train_amd.ops`; `exact` states them once more in 64 bits.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------- the cases
def _attn(name, B, Nq, Nk, H, Hkv, dh, dtype="bf16", mask="none", packed=False, bwd=False):
    return {"name": name, "op": "attn", "B": B, "Nq": Nq, "Nk": Nk, "H": H, "Hkv": Hkv, "dh": dh, "dtype": dtype, "mask": mask,
            "packed": packed, "bwd": bwd}


def _rope(name, B, N, H, dh, axes, dtype="bf16", prefix=0, interleaved=False, inverse=False, two=False, own_pos=False, span=64):
    return {"name": name, "op": "rope", "B": B, "N": N, "H": H, "dh": dh, "axes": axes, "dtype": dtype, "prefix": prefix,
            "interleaved": interleaved, "inverse": inverse, "two": two, "own_pos": own_pos, "span": span}


def _topk(name, rows, K, k, dtype="f32", ddtype="bf16", tail=False, weights=False):
    return {"name": name, "op": "topk", "rows": rows, "K": K, "k": k, "dtype": dtype, "ddtype": ddtype, "tail": tail, "weights": weights}


def listed():
    return [
        # one new query against one image's 197 tokens: a single step of a decoder, all latency
        _attn("attn-one-query", 1, 1, 197, 12, 12, 64),
        # attentive pooling of a batch at 518^2 / 14 (1370 tokens) by one learned query, keys and values packed by one projection
        _attn("attn-pool", 64, 1, 1370, 12, 12, 64, packed=True),
        # 100 object queries against a padded batch (lengths differ, one image is empty, some tokens are dropped)
        _attn("attn-decoder-padded", 16, 100, 1025, 8, 8, 64, dtype="f16", mask="both"),
        # a video memory of 32 frames of 28 x 28 tokens read by one frame's queries, four query heads a key head
        _attn("attn-video-memory", 2, 784, 25088, 16, 4, 128),
        # a predictor of 196 masked tokens trained against the encoder's 1370
        _attn("attn-train", 32, 196, 1370, 12, 12, 64, packed=True, bwd=True),
        # training an attentive pooling head on a padded batch
        _attn("attn-pool-train", 64, 1, 785, 6, 6, 64, mask="lens", bwd=True),
        # 8 frames and their class token against the video they come from: the long training case, shared key heads, odd sizes
        _attn("attn-video-train", 2, 1569, 6273, 16, 8, 64, mask="mask", bwd=True),
        # one token a sequence at its own (t, h, w): serving
        _rope("rope-one-token", 16, 1, 12, 64, 3, own_pos=True, span=100000),
        # 8 x 14 x 14 video tokens behind a class token, q and k of a packed projection in one call
        _rope("rope-video", 16, 1569, 12, 64, 3, prefix=1, two=True, span=32),
        # gradient (inverse rotation) of a batch of dropped-token images, interleaved pairs, positions per sample, odd count, 32 bits
        _rope("rope-grad", 32, 1025, 16, 128, 2, dtype="f32", interleaved=True, inverse=True, own_pos=True, span=512),
        # classification heads: 1000 classes, the teacher's ten best, the rest in one bucket
        _topk("topk-classes", 256, 1000, 10, ddtype="f32", tail=True),
        # prototype rows of a step's crops: 65 536 prototypes, 256 kept of the frozen teacher's
        _topk("topk-prototypes", 2048, 65536, 256, tail=True, weights=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "rope", "topk"])
    while True:
        if op == "attn":
            bwd = rng.random() < 0.5
            dh = rng.choice([32, 64, 64, 72, 80, 128])
            Hkv, g = rng.choice([1, 2, 3, 4, 6, 8, 12]), rng.choice([1, 1, 2, 4])
            c = _attn("", _log(rng, 1, 64), 1 if rng.random() < 0.3 else _log(rng, 1, 2048), _log(rng, 1, 26000), Hkv * g, Hkv, dh,
                      rng.choice(["bf16", "f16"]), rng.choice(["none", "lens", "mask", "both"]), rng.random() < 0.5, bwd)
        elif op == "rope":
            c = _rope("", _log(rng, 1, 64), 1 if rng.random() < 0.2 else _log(rng, 1, 6272), rng.choice([3, 6, 8, 12, 16]),
                      rng.choice([32, 64, 64, 80, 128]), rng.choice([1, 2, 3, 4]), rng.choice(["bf16", "f16", "f32"]), 0, rng.random() < 0.5,
                      rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5, _log(rng, 16, 1000000))
            c["prefix"] = rng.choice([0, 0, 1, 5]) if c["N"] > 5 else 0
        else:
            K = _log(rng, 10, 140000)
            dt = rng.choice(["f32", "bf16", "f16"])
            c = _topk("", _log(rng, 1, 8192), K, min(K, _log(rng, 1, 512)), dt, rng.choice(["f32", "bf16"]) if dt == "f32" else dt,
                      rng.random() < 0.5, rng.random() < 0.5)
            c["k"] = max(1, min(c["k"], K // 2))
        w, top = work(c), [work(x) for x in listed() if x["op"] == op]
        kv = c["B"] * c["H"] * c["Nk"] * c["dh"] if op == "attn" else 0
        if w["bytes"] <= max(x["bytes"] for x in top) and w["flops"] <= max(x["flops"] for x in top) and kv <= 1 << 29:
            del c["name"]
            return c


def work(case):
    c = case
    if c["op"] == "attn":
        q, kv = c["B"] * c["Nq"] * c["H"] * c["dh"], c["B"] * c["Nk"] * c["Hkv"] * c["dh"]
        b = 2 * (2 * q + 2 * kv) + 4 * c["B"] * c["Nq"] * c["H"]
        f = 4 * q * c["Nk"]
        if c["bwd"]:    # dout in as well; dq, dk and dv out
            b += 2 * (2 * q + 2 * kv)
            f += 10 * q * c["Nk"]
        b += c["B"] * c["Nk"] * (c["mask"] in ("mask", "both")) + 4 * c["B"] * (c["mask"] in ("lens", "both"))
        return {"bytes": b, "flops": f}
    if c["op"] == "rope":
        n = c["B"] * c["N"] * c["H"] * c["dh"] * (2 if c["two"] else 1)
        pos = (c["B"] if c["own_pos"] else 1) * (c["N"] - c["prefix"]) * c["axes"]
        return {"bytes": 2 * n * (4 if c["dtype"] == "f32" else 2) + 4 * pos, "flops": 3 * n}
    n = c["rows"] * c["K"]
    b = n * ((4 if c["dtype"] == "f32" else 2) + (4 if c["ddtype"] == "f32" else 2))
    return {"bytes": b + c["rows"] * (12 * c["k"] + 4 + 4 * c["tail"] + 4 * c["weights"]), "flops": 6 * n}


# ---------------------------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    c = dict(case)
    s = {"case": c}
    if c["op"] == "attn":
        B, Nq, Nk, H, Hkv, dh, dt = c["B"], c["Nq"], c["Nk"], c["H"], c["Hkv"], c["dh"], TYPES[c["dtype"]]
        s["q"] = (randn(B, Nq, H, dh) * 1.5).to(dt)
        if c["packed"]:
            kv = randn(B, Nk, 2, Hkv, dh).to(dt)
            s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        else:
            s["k"], s["v"] = randn(B, Nk, Hkv, dh).to(dt), randn(B, Nk, Hkv, dh).to(dt)
        s["scale"], s["lens"], s["mask"] = dh ** -0.5, None, None
        seen = torch.ones(B, Nk, dtype=torch.bool, device="cuda")
        if c["mask"] in ("lens", "both"):
            s["lens"] = torch.randint(Nk // 2, Nk + 1, (B,), device="cuda", generator=g).int()
            if B > 2:
                s["lens"][B // 2] = 0            # an image without tokens
            seen &= torch.arange(Nk, device="cuda")[None] < s["lens"][:, None]
        if c["mask"] in ("mask", "both"):
            s["mask"] = torch.rand(B, Nk, device="cuda", generator=g) < 0.8
            seen &= s["mask"]
        if c["mask"] != "none":                  # what a padded batch holds behind its tokens: anything
            s["k"][~seen] = float("nan")
            s["v"][~seen] = float("inf")
        if c["bwd"]:
            s["dout"] = randn(B, Nq, H, dh).to(dt)
        return s
    if c["op"] == "rope":
        B, N, H, dh, A, dt = c["B"], c["N"], c["H"], c["dh"], c["axes"], TYPES[c["dtype"]]
        x = randn(B, N, 2 if c["two"] else 1, H, dh).to(dt)
        s["x"], s["x2"] = x[:, :, 0], (x[:, :, 1] if c["two"] else None)
        shape = (B, N - c["prefix"], A) if c["own_pos"] else (N - c["prefix"], A)
        s["pos"] = torch.randint(0, c["span"], shape, device="cuda", generator=g, dtype=torch.int32)
        # the pairs are dealt to the axes in runs; within a run the frequencies fall from 1 to 1 / 10000; what is left over is not rotated
        half = dh // 2
        run = half // A
        i = torch.arange(half)
        s["freqs"] = torch.where(i < run * A, 10000.0 ** (-(i % run).double() / run), torch.zeros((), dtype=torch.float64)).float().cuda()
        s["axis"] = torch.where(i < run * A, i // run, torch.tensor(-1)).int().cuda()
        return s
    rows, K, k = c["rows"], c["K"], c["k"]
    z = randn(rows, K) * 2
    t = z * 0.5 + randn(rows, K) * 2
    s["inv_temp"], s["coef"] = 0.5, 1.0 / rows
    s["z"] = z.to(TYPES[c["dtype"]])
    s["t_lse"] = torch.logsumexp(t.double() * s["inv_temp"], 1).float() if c["tail"] else None
    s["t_val"], s["t_idx"] = torch.topk(t, k, dim=1)
    gone = torch.rand(rows, k, device="cuda", generator=g) < 0.05       # rows for which fewer entries were kept, one without any
    if rows > 2:
        gone[rows // 2] = True
    s["t_idx"] = torch.where(gone, torch.tensor(-1, device="cuda"), s["t_idx"])
    s["weight"] = torch.rand(rows, device="cuda", generator=g) + 0.5 if c["weights"] else None
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    return {"attn": _run_attn, "rope": _run_rope, "topk": _run_topk}[state["case"]["op"]](state)


def _seen(s):
    """[B, Nk] truth values of the visible keys, None where all are."""
    B, Nk = s["case"]["B"], s["case"]["Nk"]
    seen = None
    if s["lens"] is not None:
        seen = torch.arange(Nk, device="cuda")[None] < s["lens"][:, None]
    if s["mask"] is not None:
        seen = s["mask"] if seen is None else seen & s["mask"]
    return seen


def _run_attn(s):
    c = s["case"]
    B, Nq, Nk, H, Hkv, dh, dt = c["B"], c["Nq"], c["Nk"], c["H"], c["Hkv"], c["dh"], TYPES[c["dtype"]]
    if own:
        from lightly_train_amd import ops

        if "out" not in s:      # buffers that a training or serving loop keeps from step to step
            s["out"], s["lse"] = torch.empty(B, Nq, H, dh, device="cuda", dtype=dt), torch.empty(B, H, Nq, device="cuda")
            n = ops.cross_attention_fwd_ws_floats(B, Nq, Nk, H, Hkv, dh)
            if c["bwd"]:
                n = max(n, ops.cross_attention_bwd_ws_floats(B, Nq, Nk, H, Hkv, dh))
                s["dq"] = torch.empty(B, Nq, H, dh, device="cuda", dtype=dt)
                dkv = torch.empty(B, Nk, 2, Hkv, dh, device="cuda", dtype=dt)
                s["dk"], s["dv"] = (dkv[:, :, 0], dkv[:, :, 1]) if c["packed"] else (dkv.view(2, B, Nk, Hkv, dh)[0], dkv.view(2, B, Nk, Hkv, dh)[1])
            s["ws"] = torch.empty(n, device="cuda")
        ops.cross_attention_fwd(s["q"], s["k"], s["v"], s["out"], s["lse"], s["scale"], key_lens=s["lens"], key_mask=s["mask"], ws=s["ws"])
        if not c["bwd"]:
            return s["out"], s["lse"]
        ops.cross_attention_bwd(s["q"], s["k"], s["v"], s["out"], s["dout"], s["lse"], s["dq"], s["dk"], s["dv"], s["scale"],
                                key_lens=s["lens"], key_mask=s["mask"], ws=s["ws"])
        return s["out"], s["lse"], s["dq"], s["dk"], s["dv"]
    G = H // Hkv
    seen = _seen(s)
    q = s["q"].float().view(B, Nq, Hkv, G, dh).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Nq, dh)
    k, v = (s[n].float() if seen is None else torch.where(seen[:, :, None, None], s[n].float(), 0.0) for n in ("k", "v"))
    k, v = k.permute(0, 2, 1, 3).contiguous(), v.permute(0, 2, 1, 3).contiguous()       # [B, Hkv, Nk, dh]
    z = torch.matmul(q, k.transpose(2, 3)) * s["scale"]                                  # [B, Hkv, G Nq, Nk]
    if seen is not None:
        z = z.masked_fill(~seen[:, None, None, :], -math.inf)
    top = z.amax(3, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(z - top)
    total = p.sum(3, keepdim=True)
    lse = torch.log(total) + torch.where(total > 0, top, 0.0)
    p = p / torch.where(total > 0, total, 1.0)
    o = torch.matmul(p, v)

    def rows(x):        # [B, Hkv, G Nq, dh] -> [B, Nq, H, dh]
        return x.view(B, Hkv, G, Nq, dh).permute(0, 3, 1, 2, 4).reshape(B, Nq, H, dh).to(dt)

    res = rows(o), lse.view(B, H, Nq)
    if not c["bwd"]:
        return res
    do = s["dout"].float().view(B, Nq, Hkv, G, dh).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Nq, dh)
    dv = torch.matmul(p.transpose(2, 3), do)
    dz = p * (torch.matmul(do, v.transpose(2, 3)) - (do * o).sum(3, keepdim=True)) * s["scale"]
    dq, dk = torch.matmul(dz, k), torch.matmul(dz.transpose(2, 3), q)
    return (*res, rows(dq), dk.permute(0, 2, 1, 3).to(dt), dv.permute(0, 2, 1, 3).to(dt))


def _run_rope(s):
    c = s["case"]
    x, x2, N, dh, n0 = s["x"], s["x2"], c["N"], c["dh"], c["prefix"]
    if own:
        from lightly_train_amd import ops

        if "out" not in s:
            s["out"] = torch.empty(x.shape, device="cuda", dtype=x.dtype)
            s["out2"] = torch.empty(x.shape, device="cuda", dtype=x.dtype) if x2 is not None else None
        ops.rope_axes(x, s["out"], s["pos"], s["freqs"], s["axis"], prefix=n0, interleaved=c["interleaved"], inverse=c["inverse"], x2=x2, out2=s["out2"])
        return (s["out"],) if x2 is None else (s["out"], s["out2"])
    ax = s["axis"].long()
    turn = s["pos"].double()[..., ax.clamp(min=0)] * torch.where(ax >= 0, s["freqs"], 0.0).double()
    if turn.dim() == 2:
        turn = turn[None]
    cos, sin = torch.cos(turn).float()[:, :, None], torch.sin(turn).float()[:, :, None]     # [B or 1, N - prefix, 1, dh / 2]
    if c["inverse"]:
        sin = -sin
    res = []
    for y in (x, x2):
        if y is None:
            continue
        z = y[:, n0:].float()
        a, b = (z[..., 0::2], z[..., 1::2]) if c["interleaved"] else (z[..., : dh // 2], z[..., dh // 2:])
        ra, rb = a * cos - b * sin, b * cos + a * sin
        z = torch.stack((ra, rb), -1).flatten(3) if c["interleaved"] else torch.cat((ra, rb), -1)
        res.append(torch.cat((y[:, :n0], z.to(y.dtype)), 1))
    return tuple(res)


def _run_topk(s):
    c = s["case"]
    rows, K, it = c["rows"], c["K"], s["inv_temp"]
    if own:
        from lightly_train_amd import ops

        if "d" not in s:
            s["d"], s["loss"] = torch.empty(rows, K, device="cuda", dtype=TYPES[c["ddtype"]]), torch.empty(rows, device="cuda")
        ops.topk_kl_fwd_bwd(s["z"], s["t_val"], s["t_idx"], it, s["coef"], s["loss"], s["d"], t_lse=s["t_lse"], row_weight=s["weight"])
        return s["loss"], s["d"]
    here = s["t_idx"] >= 0
    some = here.any(1, keepdim=True)
    at = s["t_idx"].clamp(min=0)
    t = torch.where(here, s["t_val"].double() * it, -math.inf)
    if c["tail"]:
        p = torch.exp(t - s["t_lse"].double()[:, None])
        rest = (1.0 - p.sum(1, keepdim=True)).clamp(min=0.0)
        rest, p = rest.float(), p.float()
    else:
        t = t - torch.where(some, t.amax(1, keepdim=True), 0.0)
        e = torch.exp(t)
        p = (e / torch.where(some, e.sum(1, keepdim=True), 1.0)).float()
    z = s["z"].float() * it
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    q = e / total
    chosen = torch.gather(z, 1, at) - torch.log(total)
    loss = torch.where(p > 0, p * (torch.log(p) - chosen), 0.0).sum(1)
    w = s["coef"] * (s["weight"] if s["weight"] is not None else torch.ones(rows, device="cuda"))
    w = torch.where(some[:, 0], w, 0.0)
    dense = torch.zeros(rows, K + 1, device="cuda").scatter_(1, torch.where(here, at, K), p)[:, :K]
    if c["tail"]:
        mark = torch.zeros(rows, K + 1, device="cuda", dtype=torch.bool).scatter_(1, torch.where(here, at, K), True)[:, :K]
        q_rest = torch.where(mark, 0.0, q).sum(1, keepdim=True)
        ok = (rest > 0) & (q_rest > 0)
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - torch.log(q_rest)), 0.0)[:, 0]
        d = torch.where(mark, q - dense, q - q * torch.where(ok, rest / q_rest, 0.0))
    else:
        d = q - dense
    loss = torch.where(some[:, 0], loss, 0.0)
    return loss * w, (d * (w * it)[:, None]).to(TYPES[c["ddtype"]])


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "rope": _exact_rope, "topk": _exact_topk}[case["op"]](s)


def _exact_attn(s):
    c = s["case"]
    B, Nq, Nk, H, Hkv, dh = c["B"], c["Nq"], c["Nk"], c["H"], c["Hkv"], c["dh"]
    seen, G = _seen(s), H // Hkv
    out, lse = torch.zeros(B, Nq, H, dh, device="cuda", dtype=torch.float64), torch.full((B, H, Nq), -math.inf, device="cuda", dtype=torch.float64)
    dq = torch.zeros_like(out)
    dk, dv = (torch.zeros(B, Nk, Hkv, dh, device="cuda", dtype=torch.float64) for _ in range(2))
    for b in range(B):      # sequence by sequence, head by head, the visible keys alone
        at = torch.arange(Nk, device="cuda") if seen is None else seen[b].nonzero()[:, 0]
        if at.numel() == 0:
            continue
        for h in range(H):
            q, k, v = s["q"][b, :, h].double(), s["k"][b, at, h // G].double(), s["v"][b, at, h // G].double()
            z = (q @ k.t().contiguous()) * s["scale"]
            lse[b, h] = torch.logsumexp(z, 1)
            p = torch.exp(z - lse[b, h][:, None])
            out[b, :, h] = p @ v
            if c["bwd"]:
                do = s["dout"][b, :, h].double()
                dp = do @ v.t().contiguous()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * s["scale"]
                dq[b, :, h] = ds @ k
                dk[b, at, h // G] += ds.t().contiguous() @ q
                dv[b, at, h // G] += p.t().contiguous() @ do
    return (out, lse, dq, dk, dv) if c["bwd"] else (out, lse)


def _exact_rope(s):
    c = s["case"]
    n0, half = c["prefix"], c["dh"] // 2
    angle = torch.zeros(*s["pos"].shape[:-1], half, device="cuda", dtype=torch.float64)
    for i in range(half):
        a = int(s["axis"][i])
        if a >= 0:
            angle[..., i] = s["pos"][..., a].double() * float(s["freqs"][i])
    w = torch.polar(torch.ones_like(angle), -angle if c["inverse"] else angle).unsqueeze(-2)
    res = []
    for y in (s["x"], s["x2"]):
        if y is None:
            continue
        z = y.double().clone()
        if c["interleaved"]:
            r = torch.view_as_complex(z[:, n0:].unflatten(-1, (half, 2)).contiguous()) * w
            z[:, n0:] = torch.view_as_real(r).flatten(-2)
        else:
            r = torch.complex(z[:, n0:, :, :half], z[:, n0:, :, half:]) * w
            z[:, n0:, :, :half], z[:, n0:, :, half:] = r.real, r.imag
        res.append(z)
    return tuple(res)


def _exact_topk(s):
    c = s["case"]
    rows, K, it = c["rows"], c["K"], s["inv_temp"]
    loss = torch.zeros(rows, device="cuda", dtype=torch.float64)
    d = torch.zeros(rows, K, device="cuda", dtype=torch.float64)
    for r0 in range(0, rows, 256):      # a few rows at a time: log-probabilities, then the gradient of the bucketed divergence
        r = slice(r0, min(rows, r0 + 256))
        logq = torch.log_softmax(s["z"][r].double() * it, 1)
        n = logq.shape[0]
        p = torch.zeros(n, K + 1, device="cuda", dtype=torch.float64)
        idx = s["t_idx"][r]
        here = idx >= 0
        some = here.any(1)
        t = s["t_val"][r].double() * it
        norm = s["t_lse"][r].double() if c["tail"] else torch.logsumexp(t.masked_fill(~here, -math.inf), 1)
        pv = torch.where(here, torch.exp(t - norm[:, None]), 0.0)
        slot = torch.where(here, idx, K)
        p.scatter_(1, slot, pv)
        kept = torch.zeros(n, K + 1, device="cuda", dtype=torch.bool).scatter_(1, slot, True)[:, :K]
        p = p[:, :K]
        le = torch.where(p > 0, p * (torch.log(p) - logq), 0.0).sum(1)
        q = torch.exp(logq)
        g = q - p
        if c["tail"]:
            rest = (1.0 - pv.sum(1)).clamp(min=0.0)
            log_rest = torch.logsumexp(logq.masked_fill(kept, -math.inf), 1)
            le = le + torch.where(rest > 0, rest * (torch.log(rest) - log_rest), 0.0)
            g = torch.where(kept, g, q - rest[:, None] * torch.exp(logq - log_rest[:, None]))
        w = s["coef"] * (s["weight"][r].double() if s["weight"] is not None else torch.ones(n, device="cuda", dtype=torch.float64))
        w = torch.where(some, w, 0.0)
        loss[r], d[r] = torch.where(some, le, 0.0) * w, torch.where(some[:, None], g, 0.0) * (w * it)[:, None]
    return loss, d
