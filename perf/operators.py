"""Operators of the hybrid family's blocks and of batches behind a shared prefix: performance cases with plain forms.

Four kinds of case, each one pass through an operator as a forward pass calls it:

  gdn_prefill   the gated delta rule over the new rows of a packed batch of prompts, state slots advanced in place
  gdn_verify    the same for a few drafted rows per sequence, the state advanced afterwards by the accepted ones
  rope_part_kv  norm and rotation of a part of every head of [query | gate] rows, keys and values appended to the paged cache
  attn_shared   decode attention of a batch whose sequences share the pages of a long prefix

With `own` the framework's operators run, otherwise the plain forms below.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
PAGE = 64
EPS = 1e-6


# -- cases ---------------------------------------------------------------------------------------------------------------


def _prefill(name, seqs, rows, n_k, n_v, behind):
    return {"name": name, "kind": "gdn_prefill", "seqs": seqs, "rows": rows, "n_k": n_k, "n_v": n_v, "d": 128, "behind": behind}


def _verify(name, seqs, rows, n_k, n_v):
    return {"name": name, "kind": "gdn_verify", "seqs": seqs, "rows": rows, "n_k": n_k, "n_v": n_v, "d": 128}


def _rope(name, seqs, rows, ctx, heads, kv_heads, dim, rot, gated, interleaved, scaled, cache):
    return {"name": name, "kind": "rope_part_kv", "seqs": seqs, "rows": rows, "ctx": ctx, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "gated": gated, "interleaved": interleaved, "scaled": scaled, "cache": cache}


def _shared(name, seqs, rows, prefix, own_keys, heads, kv_heads, dim, gated):
    return {"name": name, "kind": "attn_shared", "seqs": seqs, "rows": rows, "prefix": prefix, "own_keys": own_keys, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "gated": gated}


def listed():
    return [
        # a short question to the dense hybrid shape: the latency of a prompt
        _prefill("prefill_37", 1, 37, 16, 48, False),
        # prompts of several users in one step of the mixture shape, half of them behind a cached prefix
        _prefill("prefill_5_ragged", 5, 900, 16, 32, True),
        # the largest chunk of one long document that an engine takes in a step
        _prefill("prefill_8192", 1, 8192, 16, 48, False),
        # one user with three drafts a step
        _verify("verify_1x4", 1, 4, 16, 32),
        # a full server with two drafts a step
        _verify("verify_32x3", 32, 3, 16, 48),
        # a decode step of a full server far into long contexts
        _rope("rope_decode_32_far", 32, 1, 200000, 24, 4, 256, 64, True, False, False, "bf16"),
        # a prompt chunk of the same heads
        _rope("rope_prompt_8190", 2, 4095, 1000, 24, 4, 256, 64, True, False, False, "bf16"),
        # whole heads, interleaved pairs slowed down for a long context, the 8-bit cache
        _rope("rope_q8_scaled_700", 3, 233, 70000, 32, 8, 128, 128, False, True, True, "q8_0"),
        # a few requests behind a short system prompt
        _shared("shared_4x500", 4, 1, 500, 60, 32, 8, 128, False),
        # a full server of the dense hybrid shape behind a long instruction
        _shared("shared_32x8192_gated", 32, 1, 8192, 300, 24, 4, 256, True),
        # questions about one long document, two rows each (a draft is verified)
        _shared("shared_61x2_20000", 61, 2, 20000, 150, 32, 8, 128, False),
        # small heads, many requests
        _shared("shared_128x2048_d64", 128, 1, 2048, 400, 16, 4, 64, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = [work(c) for c in listed()]
    most = {k: max(w[k] for w in top) for k in ("bytes", "flops")}
    while True:
        kind = rng.choice(("gdn_prefill", "gdn_verify", "rope_part_kv", "attn_shared"))
        n_k, n_v = rng.choice(((16, 48), (16, 32), (16, 24), (16, 16), (8, 16)))
        if kind == "gdn_prefill":
            c = _prefill("", _log(rng, 1, 16), _log(rng, 1, 8192), n_k, n_v, rng.random() < 0.5)
        elif kind == "gdn_verify":
            c = _verify("", _log(rng, 1, 64), rng.randint(2, 8), n_k, n_v)
        elif kind == "rope_part_kv":
            dim = rng.choice((64, 128, 256))
            heads, kv_heads = rng.choice(((24, 4), (16, 2), (32, 8), (16, 4), (6, 1), (28, 4)))
            c = _rope("", _log(rng, 1, 64), _log(rng, 1, 4096), _log(rng, 1, 200000), heads, kv_heads, dim, rng.choice((dim, dim // 2, dim // 4)),
                      rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5, rng.choice(("bf16", "bf16", "q8_0")))
        else:
            dim = rng.choice((64, 128, 128, 256, 256))
            heads, kv_heads = rng.choice(((24, 4), (16, 2), (32, 8), (16, 4), (8, 8), (28, 4)))
            c = _shared("", _log(rng, 1, 128), rng.choice((1, 1, 1, 2)), _log(rng, 64, 20000), _log(rng, 1, 1000), heads, kv_heads, dim, rng.random() < 0.5)
        del c["name"]
        w = work(c)
        if c["seqs"] * c["rows"] <= 8192 and all(w[k] <= most[k] for k in most):
            return c


def _lens(case, key, lo=1):
    """Ragged sizes of a case's sequences: up to case[key], one of them that long."""
    r = random.Random(case[key] * 131 + case["seqs"])
    n = [max(lo, int(case[key] * (0.35 + 0.65 * r.random()))) for _ in range(case["seqs"])]
    n[len(n) // 2] = case[key]
    return n


def work(case):
    k = case["kind"]
    if k in ("gdn_prefill", "gdn_verify"):
        B, n_k, n_v, d = case["seqs"], case["n_k"], case["n_v"], case["d"]
        T = sum(_lens(case, "rows")) if k == "gdn_prefill" else B * case["rows"]
        C = 2 * n_k * d + n_v * d
        resumed = B if k == "gdn_verify" else (B + 1) // 2 if case["behind"] else 0
        state = n_v * d * d * 4 + C * 3 * 4
        return {"bytes": T * 2 * (C + 2 * n_v * d + 2 * n_v) + (B + resumed) * state + C * 16, "flops": T * n_v * 6 * d * d}
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    if k == "rope_part_kv":
        T = sum(_lens(case, "rows"))
        cache = 2.0 if case["cache"] == "bf16" else 1.0 + 2.0 / 32
        return {"bytes": int(T * D * (2 * H + 2 * H + 4 * Hk + 2 * Hk * cache)), "flops": T * (H + Hk) * (4 * D + 3 * case["rot"])}
    R, keys = case["rows"], sum(_lens(case, "own_keys", case["rows"]))
    T = case["seqs"] * R
    return {"bytes": (case["prefix"] + keys) * 2 * Hk * D * 2 + T * H * D * (6 if case["gated"] else 4),
            "flops": 4 * H * D * (T * case["prefix"] + R * keys)}


# -- inputs --------------------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEVICE)


def _prepare_gdn(case, seed):
    gen = _gen(seed)
    B, n_k, n_v, d, K = case["seqs"], case["n_k"], case["n_v"], case["d"], 4

    def rnd(*s):
        return torch.randn(*s, device=DEVICE, generator=gen)

    def uni(*s):
        return torch.rand(*s, device=DEVICE, generator=gen)

    verify = case["kind"] == "gdn_verify"
    lens = [case["rows"]] * B if verify else _lens(case, "rows")
    T, C = sum(lens), 2 * n_k * d + n_v * d
    width = C + n_v * d + 2 * n_v
    buf = torch.zeros(T, (width + 63) // 64 * 64, dtype=torch.bfloat16, device=DEVICE)      # rows of the input projection's workspace
    buf[:, :width] = rnd(T, width).to(torch.bfloat16)
    # decay rates and step sizes as such layers are initialised and stay near: A in 1 .. 16, steps of 0.001 to 0.1
    step = torch.exp(uni(n_v) * math.log(100.0) + math.log(0.001))
    order = torch.randperm(B + 2, generator=torch.Generator().manual_seed(seed)).tolist()[:B]
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    resumed = [verify or (case["behind"] and i % 2 == 0) for i in range(B)]
    pos = [(1000 if resumed[i] else 0) + t for i in range(B) for t in range(lens[i])]
    s = {"case": case, "lens": lens, "resumed": resumed, "order": order, "inp": buf[:, :width], "C": C, "z_off": C, "ab_off": C + n_v * d,
         "conv_w": rnd(C, K) * 0.4, "ssm_a": -(1 + 15 * uni(n_v)), "dt_bias": torch.log(torch.expm1(step)), "norm_w": 1 + 0.1 * rnd(d),
         "conv": rnd(B + 2, C, K - 1).to(torch.bfloat16).float(), "rec": rnd(B + 2, n_v, d, d) * 0.05, "cu": _ints(cu), "positions": _ints(pos),
         "slots": _ints(order), "out": torch.zeros(T, n_v * d, dtype=torch.bfloat16, device=DEVICE)}
    if verify:
        s["accepted"] = _ints([1 + (i * 7 + seed) % case["rows"] for i in range(B)])
    return s


def _pages(seqs, n, gen_seed, first=1):
    """Shuffled page ids for `n[i]` pages of each sequence, and the number of pages a pool needs."""
    ids = list(range(first, first + sum(n)))
    random.Random(gen_seed).shuffle(ids)
    table, at = torch.zeros(seqs, max(n), dtype=torch.int32), 0
    for i, k in enumerate(n):
        table[i, :k] = torch.tensor(ids[at:at + k], dtype=torch.int32)
        at += k
    return table, first + sum(n)


def _prepare_rope(case, seed):
    gen = _gen(seed)
    B, H, Hk, D, rot = case["seqs"], case["heads"], case["kv_heads"], case["dim"], case["rot"]
    lens = _lens(case, "rows")
    T, parts = sum(lens), 2 if case["gated"] else 1
    # the caches of the sequences hold what came before; the tokens go to the pages at their end
    starts = [max(0, case["ctx"] - 777 * i) for i in range(B)]
    used = [(starts[i] + lens[i] + PAGE - 1) // PAGE - starts[i] // PAGE for i in range(B)]
    ids, n_pages = _pages(B, used, seed)
    table = torch.zeros(B, max((starts[i] + lens[i] + PAGE - 1) // PAGE for i in range(B)), dtype=torch.int32)
    for i in range(B):
        table[i, starts[i] // PAGE:starts[i] // PAGE + used[i]] = ids[i, :used[i]]
    freqs = 1e7 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if case["scaled"]:                       # slow pairs 4 times slower, fast ones as they are, a ramp between
        ramp = ((torch.log2(freqs * 32768 / (2 * math.pi))) / 5).clamp(0, 1)
        freqs = freqs * (ramp + (1 - ramp) / 4)
    rows = torch.randn(T, (H * parts + 2 * Hk) * D, device=DEVICE, generator=gen).to(torch.bfloat16)
    if case["cache"] == "bf16":
        kv = torch.zeros(n_pages, 2, Hk, PAGE, D, dtype=torch.bfloat16, device=DEVICE)
    else:
        kv = torch.zeros(n_pages, 2 * Hk * PAGE * D * 17 // 16, dtype=torch.uint8, device=DEVICE)
    return {"case": case, "rows": rows, "kv": kv, "q_out": torch.zeros(T, H, D, dtype=torch.bfloat16, device=DEVICE),
            "q_norm": 1 + 0.1 * torch.randn(D, device=DEVICE, generator=gen), "k_norm": 1 + 0.1 * torch.randn(D, device=DEVICE, generator=gen),
            "freqs": freqs.to(DEVICE), "magnitude": 1.0 + 0.1 * math.log(4.0) if case["scaled"] else 1.0,
            "positions": _ints([starts[i] + t for i in range(B) for t in range(lens[i])]),
            "seq_ids": _ints([i for i in range(B) for _ in range(lens[i])]), "table": table.to(DEVICE)}


def _prepare_shared(case, seed):
    gen = _gen(seed)
    B, R, H, Hk, D, P = case["seqs"], case["rows"], case["heads"], case["kv_heads"], case["dim"], case["prefix"]
    keys = _lens(case, "own_keys", R)
    n_pre = P // PAGE                        # whole pages of the prefix are shared, a partly filled one is every sequence's own
    shared = n_pre * PAGE
    total = [P + k for k in keys]
    ids, n_pages = _pages(B, [(n + PAGE - 1) // PAGE - n_pre for n in total], seed, 1 + n_pre)
    pre = torch.randperm(n_pre, generator=torch.Generator().manual_seed(seed)).to(torch.int32) + 1
    table = torch.cat([pre[None].expand(B, n_pre), ids], 1).contiguous()
    kv = torch.randn(n_pages, 2, Hk, PAGE, D, device=DEVICE, generator=gen).to(torch.bfloat16)
    q = torch.randn(B * R, H, D, device=DEVICE, generator=gen).to(torch.bfloat16)
    rows = torch.randn(B * R, H, 2, D, device=DEVICE, generator=gen).to(torch.bfloat16) if case["gated"] else None      # [query | gate] rows of the projection
    return {"case": case, "total": total, "shared": shared, "kv": kv, "q": q, "gate": rows[:, :, 1] if case["gated"] else None, "table": table.to(DEVICE),
            "seq_lens": _ints(total), "shared_len": _ints([shared]), "out": torch.zeros_like(q), "scale": D ** -0.5}


def prepare(case, seed):
    return {"gdn_prefill": _prepare_gdn, "gdn_verify": _prepare_gdn, "rope_part_kv": _prepare_rope, "attn_shared": _prepare_shared}[case["kind"]](case, seed)


# -- plain forms ---------------------------------------------------------------------------------------------------------


def _padded(s):
    """Row index [B, longest] of every sequence's rows and which of them there are."""
    n = torch.tensor(s["lens"], device=DEVICE)
    t = torch.arange(max(s["lens"]), device=DEVICE)
    there = t[None] < n[:, None]
    return (s["cu"][:-1, None].long() + t[None]).clamp_max(s["inp"].shape[0] - 1), there, n


def _conv_inputs(s, rows, n):
    """[old window | rows] of every sequence and the window behind its first n rows."""
    C, K = s["conv_w"].shape
    keep = torch.tensor(s["resumed"], device=DEVICE)[:, None, None]
    old = torch.where(keep, s["conv"][s["slots"].long()].transpose(1, 2), 0.0)
    x = torch.cat([old, s["inp"][:, :C].float()[rows]], 1)
    at = n.long()[:, None] + torch.arange(K - 1, device=DEVICE)[None]
    return x, torch.gather(x, 1, at[:, :, None].expand(-1, -1, C)).transpose(1, 2)


def _gdn_rows(s):
    """Of every (sequence, padded row): q, k [B, T, heads, d], v, log decay, write strength (0 behind a sequence), and the windows' inputs."""
    case = s["case"]
    n_k, n_v, d = case["n_k"], case["n_v"], case["d"]
    rows, there, n = _padded(s)
    x, window = _conv_inputs(s, rows, s["accepted"] if case["kind"] == "gdn_verify" else n)
    T, K = rows.shape[1], s["conv_w"].shape[1]
    y = torch.stack([x[:, j:j + T] * s["conv_w"][:, j] for j in range(K)]).sum(0)
    y = y / (1 + torch.exp(-y))
    q, k, v = (p.unflatten(2, (-1, d)) for p in torch.split(y, [n_k * d, n_k * d, n_v * d], 2))
    q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6) * d ** -0.5
    k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    head = torch.arange(n_v, device=DEVICE) % n_k
    ab = s["inp"][:, s["ab_off"]:].float()[rows]
    a = ab[..., :n_v] + s["dt_bias"]
    soft = torch.clamp_min(a, 0) + torch.log1p(torch.exp(-a.abs()))
    g = torch.where(there[..., None], s["ssm_a"] * soft, 0.0)
    beta = torch.where(there[..., None], 1 / (1 + torch.exp(-ab[..., n_v:])), 0.0)
    return q[:, :, head], k[:, :, head], v, g, beta, rows, there, window


def _gated_norm(s, o, rows, there):
    z = s["inp"][:, s["z_off"]:s["ab_off"]].float()[rows].view(o.shape)
    r = o / torch.sqrt((o * o).mean(-1, keepdim=True) + EPS) * s["norm_w"] * z / (1 + torch.exp(-z))
    s["out"][rows[there]] = r.flatten(2)[there].to(torch.bfloat16)


def _plain_prefill(s):
    """Chunks of 64 rows: one triangular inverse per chunk and head (all at once), then the chunks one after the other."""
    q, k, v, g, beta, rows, there, window = _gdn_rows(s)
    B, T, H, d = q.shape
    n, L = (T + 63) // 64, 64

    def cut(x):                              # [B, T, H, ...] -> [chunks, B, H, 64, ...]
        x = torch.nn.functional.pad(x.transpose(1, -1), (0, n * L - T)).transpose(1, -1)
        return x.unflatten(1, (n, L)).permute(1, 0, 3, 2, *range(4, x.dim() + 1))

    qc, kc, vc, G, b = cut(q), cut(k), cut(v), cut(g).cumsum(-1), cut(beta)
    low = torch.ones(L, L, dtype=torch.bool, device=DEVICE).tril()
    M = torch.exp(torch.where(low, G[..., :, None] - G[..., None, :], -math.inf))
    A = torch.where(low.tril(-1), kc @ kc.transpose(-1, -2) * M * b[..., None], 0.0)
    inv = torch.eye(L, device=DEVICE).expand(A.shape).clone()
    for i in range(1, L):                    # forward substitution, every chunk and head at once
        inv[..., i, :i] = -(A[..., i, None, :i] @ inv[..., :i, :i])[..., 0, :]
    P = qc @ kc.transpose(-1, -2) * M
    S = torch.where(torch.tensor(s["resumed"], device=DEVICE)[:, None, None, None], s["rec"][s["slots"].long()], 0.0)
    o = torch.empty_like(vc)
    for c in range(n):
        e = torch.exp(G[c])[..., None]
        U = inv[c] @ (b[c][..., None] * (vc[c] - e * (kc[c] @ S)))
        o[c] = e * (qc[c] @ S) + P[c] @ U
        S = torch.exp(G[c][..., -1])[..., None, None] * S + kc[c].transpose(-1, -2) @ (torch.exp(G[c][..., -1:] - G[c])[..., None] * U)
    s["rec"][s["slots"].long()] = S
    s["conv"][s["slots"].long()] = window
    _gated_norm(s, o.permute(1, 0, 3, 2, 4).flatten(1, 2)[:, :T], rows, there)
    return s["out"], s["rec"], s["conv"]


def _plain_verify(s):
    q, k, v, g, beta, rows, there, window = _gdn_rows(s)
    S = s["rec"][s["slots"].long()]
    kept, o = S, []
    for t in range(q.shape[1]):              # drafted rows, a handful
        S = S * torch.exp(g[:, t])[..., None, None]
        u = (v[:, t] - (S * k[:, t][..., None]).sum(-2)) * beta[:, t][..., None]
        S = S + k[:, t][..., None] * u[..., None, :]
        o.append((S * q[:, t][..., None]).sum(-2))
        kept = torch.where((s["accepted"] > t)[:, None, None, None], S, kept)
    s["rec"][s["slots"].long()] = kept
    s["conv"][s["slots"].long()] = window
    _gated_norm(s, torch.stack(o, 1), rows, there)
    return s["out"], s["rec"], s["conv"]


def _eight_bit(x):
    """Blocks of 32 as 8-bit numbers and their scales: the largest / 127, rounded up to seven bits behind the point."""
    b = x.unflatten(-1, (-1, 32))
    up = ((b.abs().amax(-1) * (1.0 / 127.0)).view(torch.int32) + 0xFFFF) & -65536
    sc = up.view(torch.float32).to(torch.float16)
    f = sc.float()[..., None]
    return torch.where(f > 0, torch.round(b * torch.where(f > 0, 1 / f, f)), 0.0).clamp(-127, 127).to(torch.int8).flatten(-2), sc


def _q8_parts(kv, Hk, D):
    n = 2 * Hk * PAGE * D
    return kv[:, :n].view(torch.int8).view(-1, 2, Hk, PAGE, D), kv[:, n:].view(torch.float16).view(-1, 2, Hk, PAGE, D // 32)


def _cache_values(kv, Hk, D):
    """What a cache stands for, in 16 bits."""
    if kv.dtype != torch.uint8:
        return kv
    x, sc = _q8_parts(kv, Hk, D)
    return (x.unflatten(-1, (-1, 32)).float() * sc.float()[..., None]).flatten(-2).to(torch.float16)


def _plain_rope(s):
    case, x = s["case"], s["rows"].float()
    H, Hk, D, rot = case["heads"], case["kv_heads"], case["dim"], case["rot"]
    parts, pos = 2 if case["gated"] else 1, s["positions"].long()
    T = x.shape[0]
    q, k, v = x[:, :H * D * parts].view(T, H, parts, D)[:, :, 0], x[:, H * D * parts:][:, :Hk * D].view(T, Hk, D), x[:, -Hk * D:].view(T, Hk, D)
    turn = torch.remainder(pos.double()[:, None] * s["freqs"], 2 * math.pi)
    cos, sin = (s["magnitude"] * torch.cos(turn)).float()[:, None], (s["magnitude"] * torch.sin(turn)).float()[:, None]

    def turned(x, w):
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        if case["interleaved"]:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([y, x[..., rot:]], -1)

    s["q_out"].copy_(turned(q, s["q_norm"]))
    page, off = s["table"][s["seq_ids"].long(), pos // PAGE].long(), pos % PAGE
    for i, y in enumerate((turned(k, s["k_norm"]), v)):
        if case["cache"] == "bf16":
            s["kv"][page, i, :, off] = y.to(torch.bfloat16)
        else:
            eight, sc = _eight_bit(y.contiguous())
            data, scales = _q8_parts(s["kv"], Hk, D)
            data[page, i, :, off] = eight
            scales[page, i, :, off] = sc
    return s["q_out"], _cache_values(s["kv"], Hk, D)


def _plain_shared(s):
    """The shared pages once for all rows, the rest of every sequence padded to the longest, one softmax over both."""
    case, kv = s["case"], s["kv"]
    B, R, H, Hk, D, n_pre = case["seqs"], case["rows"], case["heads"], case["kv_heads"], case["dim"], s["shared"] // PAGE
    G = H // Hk
    q = s["q"].float().view(B, R, Hk, G, D).permute(2, 0, 3, 1, 4) * s["scale"]                  # [Hk, B, G, R, D]
    pre = kv[s["table"][0, :n_pre].long()].float().permute(1, 2, 0, 3, 4).flatten(2, 3)
    tail = kv[s["table"][:, n_pre:].long()].float().permute(2, 3, 0, 1, 4, 5).flatten(3, 4)
    a = (q.reshape(Hk, -1, D) @ pre[0].transpose(1, 2)).view(Hk, B, G * R, -1)
    b = q.reshape(Hk, B, G * R, D) @ tail[0].transpose(2, 3)
    key = s["shared"] + torch.arange(b.shape[-1], device=DEVICE)
    last = s["seq_lens"][:, None] - R + torch.arange(R, device=DEVICE)                           # position of every row
    dead = key[None, None] > last[..., None]
    b = torch.where(dead[:, None].expand(B, G, R, -1).reshape(1, B, G * R, -1), -math.inf, b)
    top = torch.maximum(b.amax(-1, keepdim=True), a.amax(-1, keepdim=True)) if n_pre else b.amax(-1, keepdim=True)
    a, b = torch.exp(a - top), torch.exp(b - top)
    o = (a.flatten(1, 2) @ pre[1]).view(Hk, B, G * R, D) + b @ tail[1]
    o = o / (a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True))
    o = o.view(Hk, B, G, R, D).permute(1, 3, 0, 2, 4).reshape(B * R, H, D)
    if s["gate"] is not None:
        o = o / (1 + torch.exp(-s["gate"].float()))
    s["out"].copy_(o)
    return s["out"]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return {"gdn_prefill": _plain_prefill, "gdn_verify": _plain_verify, "rope_part_kv": _plain_rope, "attn_shared": _plain_shared}[kind](s)
    from llaminar_b200 import ops
    if kind == "gdn_prefill":
        ops.gdn_prefill(s["inp"], s["C"], s["z_off"], s["ab_off"], s["conv_w"], s["ssm_a"], s["dt_bias"], s["norm_w"], s["conv"], s["rec"],
                        s["positions"], s["cu"], s["slots"], s["out"], case["n_k"], 0, EPS)
        return s["out"], s["rec"], s["conv"]
    if kind == "gdn_verify":
        stash = ops.gdn_verify(s["inp"], s["C"], s["z_off"], s["ab_off"], s["conv_w"], s["ssm_a"], s["dt_bias"], s["norm_w"], s["conv"], s["rec"],
                               s["slots"], s["out"], case["n_k"], 0, EPS)
        ops.gdn_commit(stash, s["accepted"], s["conv"], s["rec"])
        return s["out"], s["rec"], s["conv"]
    if kind == "rope_part_kv":
        ops.rope_part_kv(s["rows"], s["q_out"], s["kv"], s["q_norm"], s["k_norm"], s["freqs"], s["magnitude"], s["positions"], s["seq_ids"], s["table"],
                         case["heads"], case["kv_heads"], case["dim"], EPS, gated=case["gated"], interleaved=case["interleaved"])
        return s["q_out"], _cache_values(s["kv"], case["kv_heads"], case["dim"])
    ops.attn_decode_shared(s["q"], s["kv"], s["out"], s["table"], s["seq_lens"], s["shared_len"], case["heads"], case["kv_heads"], case["dim"], case["rows"],
                           s["scale"], ops.scratch_for(s["q"].device), gate=s["gate"], max_shared=s["shared"])
    return s["out"]


# -- results in 64 bits --------------------------------------------------------------------------------------------------


def _exact_gdn(s):
    """Token after token, all sequences side by side."""
    case = s["case"]
    n_k, n_v, d, lens = case["n_k"], case["n_v"], case["d"], s["lens"]
    first, slots, w = s["cu"].tolist(), s["order"], s["conv_w"].double()
    verify = case["kind"] == "gdn_verify"
    take = s["accepted"].tolist() if verify else lens
    rec, conv = s["rec"].double().clone(), s["conv"].double().clone()
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEVICE)
    B, kd = len(lens), n_k * d
    live = torch.tensor(s["resumed"], device=DEVICE).double()
    S, win = rec[slots] * live[:, None, None, None], conv[slots] * live[:, None, None]
    end, end_win = S.clone(), win.clone()
    key_head = [h % n_k for h in range(n_v)]
    for t in range(max(lens)):
        who = [i for i in range(B) if t < lens[i]]
        at = torch.tensor([first[i] + t for i in who], device=DEVICE)
        ix = torch.tensor(who, device=DEVICE)
        row = s["inp"][at].double()
        old = win[ix]
        new = torch.cat([old, row[:, :s["C"], None]], 2)
        y = (new * w).sum(2)
        y = y * torch.sigmoid(y)
        qk = y[:, :2 * kd].view(-1, 2, n_k, d)
        qk = qk * torch.rsqrt(qk.square().sum(-1, keepdim=True) + 1e-6)
        q, k = qk[:, 0][:, key_head] / math.sqrt(d), qk[:, 1][:, key_head]
        v = y[:, 2 * kd:].view(-1, n_v, d)
        ab = row[:, s["ab_off"]:]
        decay = torch.exp(s["ssm_a"].double() * torch.nn.functional.softplus(ab[:, :n_v] + s["dt_bias"].double(), threshold=1e9))
        X = S[ix] * decay[..., None, None]
        u = torch.sigmoid(ab[:, n_v:])[..., None] * (v - (k.unsqueeze(2) @ X).squeeze(2))
        X = X + k.unsqueeze(3) @ u.unsqueeze(2)
        o = (q.unsqueeze(2) @ X).squeeze(2)
        z = row[:, s["z_off"]:s["ab_off"]].view(o.shape)
        out[at] = (o * torch.rsqrt(o.square().mean(-1, keepdim=True) + EPS) * s["norm_w"].double() * z * torch.sigmoid(z)).flatten(1)
        S[ix], win[ix] = X, new[:, :, 1:]
        done = [i for i in who if t + 1 == take[i]]
        end[done], end_win[done] = S[done], win[done]
    rec[slots], conv[slots] = end, end_win
    return out, rec, conv


def _exact_rope(s):
    case = s["case"]
    H, Hk, D, rot = case["heads"], case["kv_heads"], case["dim"], case["rot"]
    per = 2 if case["gated"] else 1
    x = s["rows"].double().view(-1, H * per + 2 * Hk, D)
    pos = s["positions"].long()
    ang = pos.double().unsqueeze(1) * s["freqs"]
    spin = torch.polar(torch.full_like(ang, s["magnitude"]), ang).unsqueeze(1)
    order = torch.arange(rot, device=DEVICE).view(-1, 2) if case["interleaved"] else torch.arange(rot, device=DEVICE).view(2, -1).t()

    def rotated(h, w):
        h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * w.double()
        y = torch.view_as_real(torch.complex(h[..., order[:, 0]], h[..., order[:, 1]]) * spin)
        h[..., order[:, 0]], h[..., order[:, 1]] = y[..., 0], y[..., 1]
        return h

    q, k, v = rotated(x[:, :H * per:per].clone(), s["q_norm"]), rotated(x[:, H * per:H * per + Hk].clone(), s["k_norm"]), x[:, H * per + Hk:]
    pages = torch.zeros(s["kv"].shape[0], 2, Hk, PAGE, D, dtype=torch.float64, device=DEVICE)
    at = s["table"][s["seq_ids"].long(), torch.div(pos, PAGE, rounding_mode="floor")].long()
    pages[at, 0, :, pos % PAGE], pages[at, 1, :, pos % PAGE] = k, v
    # an 8-bit cache stands for values that the rounding decides: no exact value
    return q, pages if case["cache"] == "bf16" else None


def _exact_shared(s):
    case = s["case"]
    R, H, Hk, D = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEVICE)
    for i, n in enumerate(s["total"]):
        pages = s["table"][i, :(n + PAGE - 1) // PAGE].long()
        K, V = (s["kv"][pages, j].double().transpose(0, 1).flatten(1, 2)[:, :n].repeat_interleave(H // Hk, 0) for j in (0, 1))
        q = s["q"][i * R:(i + 1) * R].double().transpose(0, 1)
        sc = q @ K.transpose(1, 2) * s["scale"]
        see = torch.arange(n, device=DEVICE)[None] <= torch.arange(n - R, n, device=DEVICE)[:, None]
        out[i * R:(i + 1) * R] = (torch.softmax(sc.masked_fill(~see, -math.inf), -1) @ V).transpose(0, 1)
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())


def exact(case, seed):
    s = prepare(case, seed)
    return {"gdn_prefill": _exact_gdn, "gdn_verify": _exact_gdn, "rope_part_kv": _exact_rope, "attn_shared": _exact_shared}[case["kind"]](s)
