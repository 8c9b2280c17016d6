"""The operators of the 8-bit key/value cache, as cases that can be timed and compared: appending tokens to it, causal attention over it
(prompts, portions, single tokens, with the attention weights that every cached token received), and evicting tokens by those weights.

The cache holds E4M3 numbers with a scale for each block of tokens and kv head.  With s a block's scale, a number x is held as
e4m3(x / s) and stands for s times that.  Scales are powers of two: the smallest with |x| <= 448 s for all the block's numbers.

``own`` false: the operators in plain torch; true: the framework's calls.  ``exact()`` is the definition in 64 bits, written by itself.
"""
import math

import torch

own = False

BF16, F32, F64, F8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
TYPES = {"bf16": BF16, "f32": F32}
DEV = "cuda"


def listed():
    return [
        # ---- append
        # the new token of one sequence of a small model: a launch's latency
        dict(name="append_1_token", op="append", dtype="bf16", n=1, kv_heads=8, dim=128, vdim=128, block=64, pos=600, len=1, ragged=False),
        # the new tokens of a served batch, each in the middle of some block, whose scale may grow
        dict(name="append_64_tokens", op="append", dtype="bf16", n=64, kv_heads=8, dim=128, vdim=128, block=32, pos=3900, len=1, ragged=True),
        # whole prompts of unequal lengths behind a prefill's projections
        dict(name="append_prompts", op="append", dtype="bf16", n=16, kv_heads=8, dim=128, vdim=128, block=64, pos=0, len=2048, ragged=True),
        # ---- attention
        # a single user on a small model: eight key heads with a few hundred tokens each
        dict(name="decode_1x700", op="attention", dtype="bf16", n=1, heads=16, kv_heads=8, dim=128, vdim=128, block=64, pos=700, len=1,
             ragged=False, softcap=0.0, extras=False, weights="none", lse=False),
        # a served batch's decode step, sequences of unequal length
        dict(name="decode_64_ragged", op="attention", dtype="bf16", n=64, heads=32, kv_heads=8, dim=128, vdim=128, block=64, pos=6000, len=1,
             ragged=True, softcap=0.0, extras=False, weights="none", lse=False),
        # few long documents, counting what attention each token receives so that the cache can be thinned out later
        dict(name="decode_4x40000_weights", op="attention", dtype="bf16", n=4, heads=32, kv_heads=8, dim=128, vdim=128, block=64, pos=40000,
             len=1, ragged=False, softcap=0.0, extras=False, weights="add", lse=False),
        # a float32 model with soft-capped scores, sinks and output gates
        dict(name="decode_f32_capped", op="attention", dtype="f32", n=8, heads=16, kv_heads=4, dim=64, vdim=64, block=32, pos=2500, len=1,
             ragged=True, softcap=20.0, extras=True, weights="none", lse=True),
        # a few drafted tokens of each sequence verified in one call
        dict(name="verify_16x5", op="attention", dtype="bf16", n=16, heads=32, kv_heads=8, dim=128, vdim=128, block=64, pos=3000, len=5,
             ragged=True, softcap=0.0, extras=False, weights="none", lse=False),
        # whole prompts
        dict(name="prompts_4x4096", op="attention", dtype="bf16", n=4, heads=32, kv_heads=8, dim=128, vdim=128, block=64, pos=0, len=4096,
             ragged=False, softcap=0.0, extras=False, weights="none", lse=False),
        # a scheduler's portions of unequal long prompts, with the weights of what they attended to
        dict(name="portions_weights", op="attention", dtype="bf16", n=5, heads=16, kv_heads=8, dim=128, vdim=128, block=32, pos=5000, len=900,
             ragged=True, softcap=0.0, extras=False, weights="last", lse=False),
        # ---- evict
        # one sequence thinned out by a few tokens
        dict(name="evict_1x700", op="evict", n=1, kv_heads=8, dim=128, vdim=128, block=64, length=700, keep=600, recent=64, ragged=False),
        # a batch of long sequences cut to half
        dict(name="evict_16x8192", op="evict", n=16, kv_heads=8, dim=128, vdim=128, block=64, length=8192, keep=4096, recent=512, ragged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "attention", "evict"])
    kv_heads, (dim, vdim) = rng.choice([1, 2, 3, 4, 8]), rng.choice([(128, 128), (128, 128), (128, 128), (64, 64), (96, 128), (80, 48)])
    case = dict(op=op, kv_heads=kv_heads, dim=dim, vdim=vdim, block=rng.choice([16, 32, 64, 64, 128]), ragged=rng.random() < 0.6)
    if op == "evict":
        length = _log(rng, 20, 16000)
        keep = max(1, int(length * rng.uniform(0.2, 1.0)))
        return dict(case, n=_log(rng, 1, max(1, min(64, 131072 // length))), length=length, keep=keep, recent=int(keep * rng.uniform(0.0, 0.6)))
    case["dtype"] = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if op == "append":
        length = rng.choice([1, _log(rng, 2, 6000)])
        return dict(case, n=_log(rng, 1, max(1, min(128, 32768 // length))), pos=rng.choice([0, _log(rng, 1, 8000)]), len=length)
    group = rng.choice([1, 2, 3, 4, 4, 8])
    kind = rng.choice(["decode", "decode", "few", "prompt"])
    if kind == "decode":
        pos, length = _log(rng, 1, 60000), 1
        n = _log(rng, 1, max(1, min(128, 250000 // pos)))
    elif kind == "few":
        pos, length = _log(rng, 1, 16000), rng.randint(2, 12)
        n = _log(rng, 1, max(1, min(32, 65536 // pos)))
    else:
        # float32 at most a few hundred rows: what a float32 model of a test or a small deployment brings
        most = 4096 if case["dtype"] == "bf16" else 500
        length = _log(rng, 13, most)
        pos = rng.choice([0, 0, _log(rng, 1, 4000)])
        n = _log(rng, 1, max(1, min(6, 2 ** 23 // (length * (pos + length)))))
    weights = rng.choice(["none", "none", "last", "add"])
    plain = rng.random() < 0.6
    return dict(case, heads=kv_heads * group, n=n, pos=pos, len=length, softcap=0.0 if plain else rng.choice([0.0, 15.0, 50.0]),
                extras=not plain, weights=weights, lse=rng.random() < 0.3)


def _lengths(case, top):
    """Lengths of the entries from the case alone: equal, or spread from about a quarter of `top` to `top`."""
    n = case["n"]
    if not case["ragged"]:
        return [top] * n
    return [max(1, top - (i * 37 + 11) % 97 * max(1, top * 3 // 4) // 97) for i in range(n)] if top > 1 else [1] * n


def entries(case):
    """(slot, position of the first token, first row, tokens) of each sequence; slots are not in the order of the rows."""
    n = case["n"]
    slots = [(i * 5 + 2) % n if n % 5 else n - 1 - i for i in range(n)]
    if case["op"] == "evict":
        return [(s, length, 0, 0) for s, length in zip(slots, _lengths(case, case["length"]))]
    at = _lengths(case, case["pos"]) if case["pos"] else [0] * n
    got, row = [], 0
    for s, p, m in zip(slots, at, _lengths(case, case["len"])):
        got.append((s, p, row, m))
        row += m
    return got


def _capacity(case):
    """Tokens a slot has room for: what is there, and some more that must stay as they are."""
    used = case["length"] if case["op"] == "evict" else case["pos"] + case["len"]
    return used + 13


def _quantised(x, block):
    """What a cache holds of x [slots, heads, tokens, dim]: E4M3 codes, and the scales [slots, heads, blocks]."""
    s, h, t, d = x.shape
    nb = -(-t // block)
    x = torch.cat([x, x.new_zeros(s, h, nb * block - t, d)], 2).view(s, h, nb, block * d)
    scale = _power(x.abs().amax(-1))
    return (x / scale[..., None]).to(F8).view(s, h, nb * block, d)[:, :, :t].contiguous(), scale


def _power(amax):
    """Smallest power of two s (not below 2^-126) with amax <= 448 s."""
    f, e = torch.frexp(amax.float())
    e = torch.where(f <= 0.875, e - 9, e - 8)
    e = torch.where(amax > 0, e, torch.full_like(e, -126)).clamp(-126, 127)
    return torch.ldexp(torch.ones_like(amax, dtype=F32), e)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)
    rnd = lambda *shape: torch.randn(*shape, generator=g, device=DEV)  # noqa: E731
    n, H, D, V, B = case["n"], case["kv_heads"], case["dim"], case["vdim"], case["block"]
    table = entries(case)
    cap, rows = _capacity(case), sum(e[3] for e in table)
    # keys have channels of their own size, as behind a norm with weights; values less so
    gain = torch.exp(0.4 * rnd(1, H, 1, D)), torch.exp(0.2 * rnd(1, H, 1, V))
    s = {"case": case, "seqs": torch.tensor(table, dtype=torch.int32, device=DEV), "entries": table}
    for name, d, w in (("k", D, gain[0]), ("v", V, gain[1])):
        codes, scales = zip(*[_quantised(rnd(1, H, cap, d) * w, B) for _ in range(n)])
        s[name], s[name + "_scale"] = torch.cat(codes), torch.cat(scales)
    s["weights"] = None
    if case["op"] == "append":
        kind = TYPES[case["dtype"]]
        # views of one fused projection's rows, as a model has them; some tokens are larger than all before them
        qkv = rnd(rows, H * (D + V)) * torch.exp(0.5 * rnd(rows, 1))
        s["qkv"] = qkv.to(kind)
        s["new_k"], s["new_v"] = s["qkv"][:, :H * D].unflatten(1, (H, D)), s["qkv"][:, H * D:].unflatten(1, (H, V))
    elif case["op"] == "attention":
        kind, heads = TYPES[case["dtype"]], case["heads"]
        s["q"] = (1.3 * rnd(rows, heads, D)).to(kind)
        s["out"] = torch.empty(rows, heads, V, dtype=kind, device=DEV)
        s["lse"] = torch.empty(rows, heads, dtype=F32, device=DEV) if case["lse"] else None
        s["sink"] = rnd(heads) if case["extras"] else None
        s["gate"] = rnd(rows, heads * V).to(kind) if case["extras"] else None
        s["scale"] = D ** -0.5
        if case["weights"] != "none":
            s["weights"] = torch.rand(n, H, cap, generator=g, device=DEV)
    else:
        # accumulated attention: a few tokens have most of it, many have none yet
        w = torch.exp(2.5 * rnd(n, H, cap))
        s["weights"] = torch.where(torch.rand(n, H, cap, generator=g, device=DEV) < 0.1, torch.zeros_like(w), w)
    if own:
        from teenygrad_b200 import ops
        s["cache"] = ops.Cache8(s["k"], s["v"], s["k_scale"], s["v_scale"], B, s["weights"])
        s["table"] = ops.step_table(table, DEV)
        if case["op"] == "attention":
            s["scratch"] = ops.cache8_attention_scratch(s["cache"], s["table"], s["q"], case["weights"] != "none")
        elif case["op"] == "evict":
            s["scratch"] = ops.cache8_evict_scratch(s["cache"], s["table"], case["keep"])
            s["kept"] = torch.empty(n, H, case["keep"], dtype=torch.int32, device=DEV)
    return s


def run(s):
    case = s["case"]
    op = case["op"]
    held = {m: s[m] for m in ("k", "v", "k_scale", "v_scale")}
    if own:
        from teenygrad_b200 import ops
        if op == "append":
            ops.cache8_append(s["cache"], s["new_k"], s["new_v"], s["table"])
            return held
        if op == "evict":
            kept = ops.cache8_evict(s["cache"], s["table"], case["keep"], case["recent"], kept=s["kept"], scratch=s["scratch"])
            return dict(held, kept=kept, weights=s["weights"])
        decay = {"none": None, "last": 0.0, "add": 0.9}[case["weights"]]
        out = ops.cache8_attention(s["q"], s["cache"], s["scale"], s["table"], softcap=case["softcap"], sink=s["sink"], gate=s["gate"],
                                   weight_decay=decay, lse=s["lse"], out=s["out"], scratch=s["scratch"])
        return {"out": out, "lse": s["lse"], "weights": s["weights"]}
    if op == "append":
        for name in ("k", "v"):
            _append(s[name], s[name + "_scale"], s["new_" + name], s["seqs"], case)
        return held
    if op == "evict":
        return dict(held, kept=_evict(s), weights=s["weights"])
    return _attention(s)


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _append(codes, scales, new, seqs, case):
    """The blocks that the new tokens fall into: new scales, what they held before at those, and the new tokens."""
    B, (cap, D) = case["block"], codes.shape[2:]
    slot, pos, row, count = (seqs[:, i].long() for i in range(4))
    most = (case["len"] + B - 2) // B + 1  # blocks that an entry can touch
    token = (pos // B * B)[:, None] + torch.arange(most * B, device=DEV)  # [n, tokens of the blocks]
    fresh = (token >= pos[:, None]) & (token < (pos + count)[:, None])
    older = token < pos[:, None]
    block = (token[:, ::B] // B).clamp(max=scales.shape[2] - 1)
    written = fresh.view(-1, most, B).any(-1)  # [n, blocks]
    x = new[(row[:, None] + token - pos[:, None]).clamp(0, new.shape[0] - 1)].float().masked_fill(~fresh[..., None, None], 0.0)
    x = x.transpose(1, 2).unflatten(2, (most, B))  # [n, heads, blocks, B, D]
    was = scales[slot[:, None], :, block].transpose(1, 2)  # [n, heads, blocks]
    had = older.view(-1, most, B).any(-1)[:, None]
    scale = _power(x.abs().amax((-1, -2)))
    scale = torch.where(had, torch.maximum(scale, was), scale)
    old = codes[slot[:, None], :, token.clamp(max=cap - 1)].transpose(1, 2).unflatten(2, (most, B)).float()
    both = torch.where(fresh.view(-1, 1, most, B, 1), x / scale[..., None, None], old * (was / scale)[..., None, None])
    both = both.flatten(2, 3).transpose(1, 2).to(F8)  # [n, tokens, heads, D]
    e, t = torch.nonzero(fresh | (older & written[:, :1]), as_tuple=True)
    codes.view(torch.uint8)[slot[e], :, token[e, t]] = both[e, t].view(torch.uint8)
    e, b = torch.nonzero(written, as_tuple=True)
    scales[slot[e], :, block[e, b]] = scale[e, :, b]


def _attention(s):
    case, seqs = s["case"], s["seqs"]
    heads, H, D, V, B = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["block"]
    G, S, L, n = heads // H, case["len"], case["pos"] + case["len"], case["n"]
    slot, pos, row, count = (seqs[:, i].long() for i in range(4))
    i, j = torch.arange(S, device=DEV), torch.arange(L, device=DEV)
    there = i < count[:, None]  # [n, S]
    rows = (row[:, None] + i).clamp(max=s["q"].shape[0] - 1)
    k = s["k"][slot, :, :L].float() * s["k_scale"][slot].repeat_interleave(B, 2)[:, :, :L, None]
    v = s["v"][slot, :, :L].float() * s["v_scale"][slot].repeat_interleave(B, 2)[:, :, :L, None]
    q = s["q"][rows].float().unflatten(2, (H, G)).permute(0, 2, 3, 1, 4).reshape(n, H, G * S, D)
    x = (q @ k.transpose(2, 3)).mul_(s["scale"]).view(n, H, G, S, L)
    if case["softcap"]:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    x.masked_fill_((j > (pos[:, None] + i)[..., None])[:, None, None], -math.inf)
    lse = torch.logsumexp(x, -1)  # [n, H, G, S]
    if case["extras"]:
        lse = torch.logaddexp(lse, s["sink"].view(H, G, 1))
    p = x.sub_(lse[..., None]).exp_()
    o = (p.view(n, H, G * S, L) @ v).view(n, H, G, S, V).permute(0, 3, 1, 2, 4)[there].reshape(-1, heads, V)
    if case["extras"]:
        o = o * torch.sigmoid(s["gate"].float()).view(-1, heads, V)
    s["out"].copy_(o)
    if case["lse"]:
        s["lse"].copy_(lse.permute(0, 3, 1, 2)[there].reshape(-1, heads))
    if case["weights"] != "none":
        got = p.masked_fill_(~there[:, None, None, :, None], 0.0).sum((2, 3))  # [n, H, L]
        live = (j < (pos + count)[:, None])[:, None]
        was = s["weights"][slot, :, :L]
        s["weights"][slot, :, :L] = torch.where(live, got if case["weights"] == "last" else 0.9 * was + got, was)
    return {"out": s["out"], "lse": s["lse"], "weights": s["weights"]}


def _evict(s):
    case, seqs = s["case"], s["seqs"]
    keep, recent, B, H, n, L = case["keep"], case["recent"], case["block"], case["kv_heads"], case["n"], case["length"]
    slot, length = seqs[:, 0].long(), seqs[:, 1].long()
    j = torch.arange(L, device=DEV)
    w = s["weights"][slot, :, :L].clone()
    w.masked_fill_((j >= (length - recent)[:, None])[:, None], math.inf)  # the last tokens stay
    w.masked_fill_((j >= length[:, None])[:, None], -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True)[1][..., :keep]  # (ties: the lowest index)
    left = torch.minimum(length, length.new_tensor(keep))
    there = (torch.arange(keep, device=DEV) < left[:, None])[:, None]
    kept = torch.sort(order.masked_fill(~there, L), -1)[0]
    there = there.expand(n, H, keep)
    at = kept.clamp(max=L - 1)
    sl, hd = slot[:, None, None], torch.arange(H, device=DEV)[None, :, None]
    nb = -(-keep // B)
    for name in ("k", "v"):
        codes, scales = s[name], s[name + "_scale"]
        x = codes[sl, hd, at].float() * scales[sl, hd, at // B][..., None]
        x.masked_fill_(~there[..., None], 0.0)
        x = torch.cat([x, x.new_zeros(n, H, nb * B - keep, x.shape[-1])], 2).unflatten(2, (nb, B))
        scale = _power(x.abs().amax((-1, -2)))
        x = (x / scale[..., None, None]).flatten(2, 3).to(F8)
        e, h, t = torch.nonzero(there, as_tuple=True)
        codes.view(torch.uint8)[slot[e], h, t] = x[e, h, t].view(torch.uint8)
        e, h, b = torch.nonzero(there[..., ::B], as_tuple=True)
        scales[slot[e], h, b] = scale[e, h, b]
    e, h, t = torch.nonzero(there, as_tuple=True)
    s["weights"][slot[e], h, t] = s["weights"][sl, hd, at][e, h, t]
    return kept.masked_fill(~there, -1).int()


# ---------------------------------------------------------------------------------------------------------------- work
def work(case):
    table = entries(case)
    H, D, V, B, n = case["kv_heads"], case["dim"], case["vdim"], case["block"], case["n"]
    blocks = lambda t: -(-t // B)  # noqa: E731
    if case["op"] == "append":
        size = 2 if case["dtype"] == "bf16" else 4
        rows = sum(e[3] for e in table)
        new = sum(blocks(p + m) - p // B for _, p, _, m in table)
        old = sum(1 for _, p, _, m in table if p % B)  # scales that are read
        return {"bytes": rows * H * (D + V) * (size + 1) + 8 * H * (new + old) + 16 * n, "flops": 3 * rows * H * (D + V)}
    if case["op"] == "evict":
        left = [min(length, case["keep"]) for _, length, _, _ in table]
        total = sum(length for _, length, _, _ in table)
        moved = sum(left)
        return {"bytes": H * (4 * total + 4 * moved + 4 * n * case["keep"] + 2 * moved * (D + V) + 8 * sum(blocks(t) for t in left)
                              + 8 * sum(blocks(length) for _, length, _, _ in table)) + 16 * n,
                "flops": 2 * moved * H * (D + V)}
    size, heads = (2 if case["dtype"] == "bf16" else 4), case["heads"]
    rows, live = sum(e[3] for e in table), sum(p + m for _, p, _, m in table)
    pairs = sum(m * p + m * (m + 1) // 2 for _, p, _, m in table)
    got = rows * heads * (D + V) * size + live * H * (D + V) + 8 * H * sum(blocks(p + m) for _, p, _, m in table) + 16 * n
    got += rows * heads * V * size + 4 * heads if case["extras"] else 0
    got += rows * heads * 4 if case["lse"] else 0
    got += {"none": 0, "last": 4, "add": 8}[case["weights"]] * live * H
    return {"bytes": got, "flops": 2 * pairs * heads * (D + V)}


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention" and case["n"] * case["heads"] * case["len"] * (case["pos"] + case["len"]) > 3e9:
        return None
    return {"append": _append64, "evict": _evict64, "attention": _attention64}[case["op"]](s)


def _code64(x):
    """The nearest E4M3 numbers to |x| <= 448, ties to even: steps of 2^(e - 3), at least 2^-9."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    e = torch.where(torch.exp2(e + 1) <= x.abs(), e + 1, torch.where((torch.exp2(e) > x.abs()) & (e > -6), e - 1, e))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _scale64(amax):
    k = torch.ceil(torch.log2((amax / 448).clamp(min=2.0 ** -126)))
    k = torch.where(448 * torch.exp2(k - 1) >= amax, k - 1, torch.where(448 * torch.exp2(k) < amax, k + 1, k))
    return torch.exp2(k.clamp(min=-126))


def _append64(s):
    got, B = {}, s["case"]["block"]
    for name in ("k", "v"):
        codes, scales, new = s[name].to(F64), s[name + "_scale"].to(F64), s["new_" + name].to(F64)
        for slot, pos, row, count in s["entries"]:
            done = pos
            while done < pos + count:
                b, end = done // B, min((done // B + 1) * B, pos + count)
                x = new[row + done - pos:row + end - pos].transpose(0, 1)  # [heads, tokens, dim]
                scale = _scale64(x.abs().amax((1, 2)))
                if done > b * B:
                    was = scales[slot, :, b].clone()
                    scale = torch.maximum(scale, was)
                    codes[slot, :, b * B:done] = _code64(codes[slot, :, b * B:done] * (was / scale)[:, None, None])
                codes[slot, :, done:end] = _code64(x / scale[:, None, None])
                scales[slot, :, b] = scale
                done = end
        got[name], got[name + "_scale"] = codes, scales
    return got


def _attention64(s):
    case = s["case"]
    H, V, B, heads = case["kv_heads"], case["vdim"], case["block"], case["heads"]
    G = heads // H
    out, lses = s["q"].new_zeros(s["q"].shape[0], heads, V, dtype=F64), torch.zeros(s["q"].shape[0], heads, dtype=F64, device=DEV)
    weights = None if s["weights"] is None else s["weights"].to(F64)
    for slot, pos, row, count in s["entries"]:
        L = pos + count
        of = torch.arange(L, device=DEV) // B
        k, v = ((s[m][slot, :, :L].to(F64) * s[m + "_scale"][slot].to(F64)[:, of, None]) for m in ("k", "v"))
        for h in range(H):
            q = s["q"][row:row + count, h * G:(h + 1) * G].to(F64)  # [count, G, D]
            x = torch.einsum("sgd,ld->sgl", q, k[h]) * s["scale"]
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            hidden = torch.arange(L, device=DEV)[None] > pos + torch.arange(count, device=DEV)[:, None]
            x.masked_fill_(hidden[:, None], -math.inf)
            top = x.amax(-1, keepdim=True)
            total = torch.exp(x - top).sum(-1, keepdim=True)
            if case["extras"]:
                total = total + torch.exp(s["sink"].to(F64)[h * G:(h + 1) * G, None] - top)
            p = torch.exp(x - top) / total
            out[row:row + count, h * G:(h + 1) * G] = torch.einsum("sgl,ld->sgd", p, v[h])
            lses[row:row + count, h * G:(h + 1) * G] = (top + torch.log(total))[..., 0]
            if weights is not None:
                w = p.sum((0, 1))
                weights[slot, h, :L] = w if case["weights"] == "last" else 0.9 * weights[slot, h, :L] + w
    if case["extras"]:
        out = out / (1 + torch.exp(-s["gate"].to(F64).view(-1, heads, V)))
    return {"out": out, "lse": lses if case["lse"] else None, "weights": weights}


def _evict64(s):
    case = s["case"]
    keep, recent, B, H = case["keep"], case["recent"], case["block"], case["kv_heads"]
    got = {m: s[m].to(F64) for m in ("k", "v", "k_scale", "v_scale", "weights")}
    for slot, length, _, _ in s["entries"]:
        if length <= keep:
            index = torch.arange(length, device=DEV).expand(H, length)
        else:
            old = s["weights"][slot, :, :length - recent]
            best = torch.sort(old.to(F64), dim=-1, descending=True, stable=True)[1][:, :keep - recent]
            last = torch.arange(length - recent, length, device=DEV).expand(H, recent)
            index = torch.cat([best.sort(-1)[0], last], 1)
        for h in range(H):
            at = index[h]
            got["weights"][slot, h, :len(at)] = got["weights"][slot, h, at].clone()
            for m in ("k", "v"):
                x = s[m][slot, h, at].to(F64) * s[m + "_scale"][slot, h, at // B].to(F64)[:, None]
                blocks = -(-len(at) // B)
                x = torch.cat([x, x.new_zeros(blocks * B - len(at), x.shape[1])]).view(blocks, -1)
                scale = _scale64(x.abs().amax(1))
                got[m][slot, h, :len(at)] = _code64(x / scale[:, None]).view(blocks * B, -1)[:len(at)]
                got[m + "_scale"][slot, h, :blocks] = scale
    return dict(got, kept=None)
