"""Timed operators of the token language models' serving path, through the framework's public entry points:

  append    keys and values of new tokens into a paged cache of 8 bits, rotated on the way (`PagedKVCache.append`, `.read`)
  attend    attention over that cache (`PagedKVCache.attend`)
  select    beam search's choice over beams and vocabulary (`beam_select`)
  reorder   the beams' states moved to where their children are, in place (`beam_reorder`)

A cache page holds 64 tokens of every key/value head: key codes [page][head][64][dim], value codes [page][head][vdim][64], and a scale for
each 16 tokens and head, [page][head][4].  A block's scale is the largest magnitude it was ever handed over the largest code (127, or 448
for e4m3); where a token makes it grow, the block's earlier codes are rounded again to the new scale.
"""
import math

import torch

own = False             # True: `run` calls the framework's operators, not their plain forms

DEV = "cuda"
PAGE, BLOCK = 64, 16
TINY = 2.0 ** -100      # a block's largest magnitude is taken as at least this
TOP = {"int8": 127.0, "e4m3": 448.0}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # one conversation's next token at a far position: what counts is the latency
        {"name": "append_1_far", "kind": "append", "seqs": 1, "rows": 1, "long": 0, "depth": 100003, "ragged": 0.0, "kv_heads": 8, "dim": 128, "vdim": 128, "codes": "int8",
         "dtype": "bf16", "rot": 128, "halves": True},
        # a full server's step: 64 sequences bring a token each, partners side by side in half of the dimensions
        {"name": "append_64", "kind": "append", "seqs": 64, "rows": 1, "long": 0, "depth": 2048, "ragged": 0.9, "kv_heads": 8, "dim": 128, "vdim": 128, "codes": "e4m3",
         "dtype": "bf16", "rot": 64, "halves": False},
        # prompts: three sequences of odd lengths, the longest 1773 tokens, behind what they already hold
        {"name": "append_prompts", "kind": "append", "seqs": 3, "rows": 1773, "long": 3, "depth": 333, "ragged": 0.5, "kv_heads": 8, "dim": 128, "vdim": 128, "codes": "int8",
         "dtype": "bf16", "rot": 128, "halves": True},
        # a long document, one user: the keys' axis is all there is to share out
        {"name": "attend_1_long", "kind": "attend", "seqs": 1, "rows": 1, "long": 0, "depth": 100003, "ragged": 0.0, "heads": 32, "kv_heads": 8, "dim": 128, "vdim": 128,
         "codes": "int8", "dtype": "bf16", "window": 0, "keep": 0, "sink": False, "rot": 128, "halves": True},
        # a full server's step of single tokens
        {"name": "attend_64", "kind": "attend", "seqs": 64, "rows": 1, "long": 0, "depth": 4096, "ragged": 0.8, "heads": 32, "kv_heads": 8, "dim": 128, "vdim": 128,
         "codes": "e4m3", "dtype": "bf16", "window": 0, "keep": 0, "sink": False, "rot": 128, "halves": True},
        # few sequences, a window that keeps the first tokens, all in fp32
        {"name": "attend_5_fp32", "kind": "attend", "seqs": 5, "rows": 1, "long": 0, "depth": 1500, "ragged": 0.9, "heads": 8, "kv_heads": 2, "dim": 128, "vdim": 128,
         "codes": "int8", "dtype": "fp32", "window": 1024, "keep": 4, "sink": True, "rot": 0, "halves": False},
        # a long prompt alone
        {"name": "attend_prompt", "kind": "attend", "seqs": 1, "rows": 4001, "long": 1, "depth": 0, "ragged": 0.0, "heads": 32, "kv_heads": 8, "dim": 128, "vdim": 128,
         "codes": "int8", "dtype": "bf16", "window": 0, "keep": 0, "sink": False, "rot": 128, "halves": True},
        # a scheduler's mixed step: two portions of prompts beside single tokens, windowed, with kept first tokens and the sink
        {"name": "attend_mixed", "kind": "attend", "seqs": 16, "rows": 331, "long": 2, "depth": 1400, "ragged": 0.6, "heads": 16, "kv_heads": 4, "dim": 128, "vdim": 128,
         "codes": "int8", "dtype": "bf16", "window": 1024, "keep": 4, "sink": True, "rot": 0, "halves": False},
        # one request searched with 4 beams
        {"name": "select_1x4", "kind": "select", "batch": 1, "beams": 4, "vocab": 32000, "dtype": "fp32", "finished": False, "penalty": 0.0},
        # a batch of 16 with 8 beams, some of them finished, ranked by the mean over the length
        {"name": "select_16x8", "kind": "select", "batch": 16, "beams": 8, "vocab": 65521, "dtype": "fp32", "finished": True, "penalty": 1.0},
        # the recurrent states of one request's 4 beams (width 1024: 8 heads of 128 x 128 in each of 6 layer runs) and their tokens
        {"name": "reorder_1x4", "kind": "reorder", "batch": 1, "beams": 4, "layers": 6, "heads": 8, "dim": 128, "vdim": 128, "tokens": 509, "dtype": "fp32"},
        # the same of 8 requests with 8 beams at width 4096
        {"name": "reorder_8x8", "kind": "reorder", "batch": 8, "beams": 8, "layers": 6, "heads": 32, "dim": 128, "vdim": 128, "tokens": 2047, "dtype": "fp32"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "select", "reorder"])
    if kind in ("append", "attend"):
        form = rng.choice(["single", "single", "mixed", "prompt"])
        dim = rng.choice([64, 80, 128, 128, 128, 192, 256])
        c = {"kind": kind, "seqs": _log(rng, 1, 64) if form != "prompt" else rng.randint(1, 2), "rows": 1, "long": 0, "ragged": round(rng.uniform(0, 0.95), 2),
             "kv_heads": rng.choice([1, 2, 3, 4, 8]), "dim": dim, "vdim": rng.choice([dim, dim, 128]), "codes": rng.choice(["int8", "e4m3"]),
             "dtype": rng.choice(["bf16", "bf16", "fp32"]), "rot": rng.choice([0, 32, 64]), "halves": rng.random() < 0.5}
        if form != "single":
            c["seqs"] = min(c["seqs"], 24)
            c["rows"] = _log(rng, 17, 400 if form == "mixed" else 1200)
            c["long"] = rng.randint(1, min(2, c["seqs"]))
        c["depth"] = _log(rng, 1, min(3 * 10 ** 8 // (c["seqs"] * c["kv_heads"] * (c["dim"] + c["vdim"])), 30000 if form == "single" else 1000))
        if kind == "attend":
            c["heads"] = c["kv_heads"] * min(rng.choice([1, 2, 4, 4, 7, 8]), 32 // c["kv_heads"])
            c["window"] = rng.choice([0, 0, _log(rng, 5, 2500)])
            c["keep"] = rng.choice([0, 1, 4, 70]) if c["window"] else 0
            c["sink"] = rng.random() < 0.3
        return c
    if kind == "select":
        return {"kind": kind, "batch": _log(rng, 1, 16), "beams": rng.choice([2, 3, 4, 5, 8, 16]), "vocab": _log(rng, 500, 30000), "dtype": rng.choice(["fp32", "fp32", "bf16"]),
                "finished": rng.random() < 0.5, "penalty": rng.choice([0.0, 0.6, 1.0])}
    return {"kind": kind, "batch": _log(rng, 1, 8), "beams": rng.choice([2, 3, 4, 5, 8]), "layers": rng.randint(1, 8), "heads": _log(rng, 1, 24), "dim": rng.choice([64, 128]),
            "vdim": rng.choice([64, 96, 128]), "tokens": _log(rng, 3, 2000), "dtype": rng.choice(["fp32", "fp32", "bf16"])}


# --------------------------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """Tokens that every sequence holds before the call, and tokens that it brings."""
    n = case["seqs"]
    past = [max(0, case["depth"] - int(case["depth"] * case["ragged"] * (e * 0.618 % 1))) for e in range(n)]
    rows = [max(1, case["rows"] - e * case["rows"] // 5) if e < case["long"] else 1 for e in range(n)]
    return past, rows


def _normal(gen, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _prepare_cache(case, gen):
    past, rows = _lengths(case)
    n, G, D, V, dtype = case["seqs"], case["kv_heads"], case["dim"], case["vdim"], DTYPES[case["dtype"]]
    held = [-(-(p + r) // PAGE) for p, r in zip(past, rows)]
    total, wide = sum(held) + 1, max(held)
    order = torch.randperm(total, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((n, wide), -1, dtype=torch.int32, device=DEV)
    first = 0
    for e, h in enumerate(held):
        table[e, :h] = order[first:first + h]
        first += h
    spread = 34.0 if case["codes"] == "int8" else 110.0     # of the codes; with the scales below, values of about one

    def codes(*shape):
        x = torch.randn(shape, generator=gen, device=DEV) * spread
        return (x.round() if case["codes"] == "int8" else x).clamp(-TOP[case["codes"]], TOP[case["codes"]]).to(CODES[case["codes"]])

    def scales():
        return (0.8 + 0.5 * torch.rand((total, G, PAGE // BLOCK), generator=gen, device=DEV)) / spread

    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    s = {"case": case, "k_codes": codes(total, G, PAGE, D), "v_codes": codes(total, G, V, PAGE), "k_scale": scales(), "v_scale": scales(), "table": table,
         "positions": ints(past), "rows": None if max(rows) == 1 else ints(starts), "most_rows": max(rows), "span": max(p + r for p, r in zip(past, rows))}
    if case["kind"] == "append":
        # keys and values as views into one projection's rows
        kv = _normal(gen, (starts[-1], G * (D + V)), dtype, 1.05)
        s["k"], s["v"] = kv[:, :G * D].unflatten(1, (G, D)), kv[:, G * D:].unflatten(1, (G, V))
        # what is read back: every token of the blocks that the call writes to
        back = [p // BLOCK * BLOCK for p in past]
        starts = [0]
        for p, b, r in zip(past, back, rows):
            starts.append(starts[-1] + p - b + r)
        s["back"], s["back_rows"], s["total_back"] = ints(back), ints(starts), starts[-1]
    else:
        H = case["heads"]
        qkv = _normal(gen, (starts[-1], H * D + G * (D + V)), dtype)
        s["q"] = qkv[:, :H * D].unflatten(1, (H, D))
    if own:
        from moshi_amd.kv_cache import PagedKVCache
        s["cache"] = PagedKVCache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"], rot_dim=case["rot"], rot_base=1e4, rot_halves=case["halves"])
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"] in ("append", "attend"):
        return _prepare_cache(case, gen)
    B, K = case["batch"], case["beams"]
    if case["kind"] == "select":
        logits = _normal(gen, (B * K, case["vocab"]), DTYPES[case["dtype"]], 3.0)
        scores = -40.0 + 2.0 * torch.randn((B, K), generator=gen, device=DEV)
        lengths = torch.randint(8, 30, (B, K), generator=gen, device=DEV, dtype=torch.int32)
        finished = torch.rand((B, K), generator=gen, device=DEV) < (0.3 if case["finished"] else -1.0)
        return {"case": case, "logits": logits, "scores": scores, "lengths": lengths, "finished": finished}
    dtype = DTYPES[case["dtype"]]
    states = [_normal(gen, (B * K, case["heads"], case["dim"], case["vdim"]), dtype) for _ in range(case["layers"])]
    states += [_normal(gen, (B * K, 3, case["heads"] * (2 * case["dim"] + case["vdim"]))) for _ in range(case["layers"])]       # the short convolutions' last inputs
    states.append(torch.randint(0, 32000, (B * K, case["tokens"]), generator=gen, device=DEV, dtype=torch.int32))
    # children of a few of the beams, best first, as a search leaves them
    parents = torch.sort((torch.rand((B, K), generator=gen, device=DEV) ** 1.5 * K).to(torch.int32).clamp(max=K - 1), dim=1).values
    return {"case": case, "states": states, "parents": parents}


# --------------------------------------------------------------------------------------------------------------------
# plain forms
# --------------------------------------------------------------------------------------------------------------------
def _rotated(x, pos, case):
    """x [rows, heads, dim] in fp32, its first `rot` dimensions turned by the angles of the rows' positions (formed in 64 bits)."""
    r = case["rot"]
    if not r:
        return x
    angle = pos.double()[:, None] * (1e4 ** (-torch.arange(0, r, 2, device=x.device, dtype=torch.float64) / r))
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if case["halves"]:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * c - b * s, a * s + b * c, x[..., r:]], dim=-1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2), x[..., r:]], dim=-1)


def _rows_of(s, positions, rows, total):
    """Sequence, position, page and place in it of every row."""
    t = torch.arange(total, device=DEV)
    if rows is None:
        seq, pos = t, positions.long()
    else:
        seq = torch.searchsorted(rows[1:].long(), t, right=True)
        pos = positions.long()[seq] + t - rows.long()[seq]
    return seq, pos, s["table"][seq, pos // PAGE].long(), pos % PAGE


def _block_update(s, x, codes, scale, transposed):
    """The blocks that x [rows, heads, n] is appended to: scales grown, earlier codes rounded again, new ones written; all in place."""
    top, n = TOP[s["case"]["codes"]], x.shape[-1]
    start = s["positions"].long()
    first = torch.arange(len(start) + 1, device=DEV) if s["rows"] is None else s["rows"].long()
    end = start + first[1:] - first[:-1]
    blocks = (s["most_rows"] + BLOCK - 2) // BLOCK + 1
    at = (start // BLOCK)[:, None] + torch.arange(blocks, device=DEV)                      # [seqs, blocks]
    pos = at[..., None] * BLOCK + torch.arange(BLOCK, device=DEV)                          # [seqs, blocks, 16]
    new = (pos >= start[:, None, None]) & (pos < end[:, None, None])
    old = pos < start[:, None, None]
    live = at * BLOCK < end[:, None]
    page = s["table"].long()[torch.arange(len(start), device=DEV)[:, None], (at * BLOCK // PAGE).clamp(max=s["table"].shape[1] - 1)]
    row = torch.where(new, first[:-1, None, None] + pos - start[:, None, None], 0)
    fresh = torch.where(new[..., None, None], x[row], 0.0)                                 # [seqs, blocks, 16, heads, n]
    part = at * BLOCK % PAGE // BLOCK
    pg, pt = page.clamp(min=0), part
    before = scale[pg, :, pt]                                                              # [seqs, blocks, heads]
    held = old[..., :1]
    grown = fresh.abs().amax(dim=(2, 4)).clamp(min=TINY) / top
    after = torch.where(held, torch.maximum(before, grown), grown)
    inv = 1.0 / after
    ratio = torch.where(held, before / after, 1.0)
    place = pos % PAGE
    earlier = (codes[pg[..., None], :, :, place] if transposed else codes[pg[..., None], :, place]).float()      # [seqs, blocks, 16, heads, n]
    fresh = (fresh * inv[:, :, None, :, None]).clamp(-top, top)
    earlier = earlier * ratio[:, :, None, :, None]
    both = torch.where(new[..., None, None], fresh, earlier)
    both = (both.round() if s["case"]["codes"] == "int8" else both).to(codes.dtype)
    put = (new | old) & live[..., None]
    if transposed:
        codes.view(torch.int8)[page[..., None].expand_as(put)[put], :, :, place[put]] = both.view(torch.int8)[put]
    else:
        codes.view(torch.int8)[page[..., None].expand_as(put)[put], :, place[put]] = both.view(torch.int8)[put]
    scale[page[live], :, part[live]] = after[live]


def _append(s):
    case = s["case"]
    k, v = s["k"].float(), s["v"].float()
    _, pos, _, _ = _rows_of(s, s["positions"], s["rows"], len(k))
    _block_update(s, _rotated(k, pos, case), s["k_codes"], s["k_scale"], False)
    _block_update(s, v, s["v_codes"], s["v_scale"], True)
    # the values that the written blocks stand for
    _, _, page, place = _rows_of(s, s["back"], s["back_rows"], s["total_back"])
    kv = s["k_codes"][page, :, place].float() * s["k_scale"][page, :, place // BLOCK][..., None]
    vv = s["v_codes"][page, :, :, place].float() * s["v_scale"][page, :, place // BLOCK][..., None]
    return kv.to(torch.bfloat16), vv.to(torch.bfloat16)


def _attend(s):
    case = s["case"]
    H, G, D, V, N = case["heads"], case["kv_heads"], case["dim"], case["vdim"], case["seqs"]
    q = s["q"].float()
    T, R, span = len(q), s["most_rows"], s["span"]
    seq, qpos, _, _ = _rows_of(s, s["positions"], s["rows"], T)
    q = _rotated(q, qpos, case)
    pages = -(-span // PAGE)
    table = s["table"][:, :pages].long()
    pg = table.clamp(min=0)
    each = lambda t: t[pg].permute(0, 2, 1, 3).reshape(N, G, pages * (PAGE // BLOCK)).repeat_interleave(BLOCK, dim=2)  # noqa: E731
    k = s["k_codes"][pg].float().permute(0, 2, 1, 3, 4).reshape(N, G, pages * PAGE, D) * each(s["k_scale"])[..., None]
    v = s["v_codes"][pg].float().permute(0, 2, 1, 4, 3).reshape(N, G, pages * PAGE, V) * each(s["v_scale"])[..., None]
    # every sequence's rows side by side, the short ones padded
    first = torch.arange(N, device=DEV) if s["rows"] is None else s["rows"][:-1].long()
    slot = torch.arange(T, device=DEV) - first[seq]
    qp = torch.zeros((N, R, G, H // G, D), device=DEV)
    qp[seq, slot] = q.unflatten(1, (G, H // G))
    scores = torch.matmul(qp.permute(0, 2, 3, 1, 4).reshape(N, G, H // G * R, D), k.transpose(2, 3).contiguous()) * D ** -0.5
    pos = (s["positions"].long()[:, None] + torch.arange(R, device=DEV))[:, None, None, :, None]          # [seqs, 1, 1, rows, 1]
    key = torch.arange(pages * PAGE, device=DEV)
    seen = key <= pos
    if case["window"]:
        seen = seen & ((key > pos - case["window"]) | (key < case["keep"]))
    seen = seen & (table >= 0).repeat_interleave(PAGE, dim=1)[:, None, None, None]
    scores = scores.view(N, G, H // G, R, -1).masked_fill(~seen, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = top.clamp(min=0.0) if case["sink"] else torch.where(top == -math.inf, 0.0, top)
    w = torch.exp(scores - top)
    total = w.sum(dim=-1, keepdim=True) + (torch.exp(-top) if case["sink"] else 0.0)
    out = torch.matmul((w / total).view(N, G, H // G * R, -1), v).view(N, G, H // G, R, V).permute(0, 3, 1, 2, 4)
    return out[seq, slot].reshape(T, H, V).to(s["q"].dtype)


def _select(s):
    case = s["case"]
    B, K, V, alpha, eos = case["batch"], case["beams"], case["vocab"], case["penalty"], 2
    x = s["logits"].double().view(B, K, V)
    top = x.amax(dim=-1, keepdim=True)
    logp = x - top - torch.exp(x - top).sum(dim=-1, keepdim=True).log()
    done = s["finished"]
    score = s["scores"].double()
    total = score[..., None] + logp
    token = torch.arange(V, device=DEV)
    total = torch.where(done[..., None], torch.where(token == eos, score[..., None], -math.inf), total)
    length = s["lengths"] + (~done).int()
    rank = (total / length.double().pow(alpha)[..., None]).flatten(1)
    at = torch.sort(rank, dim=1, descending=True, stable=True).indices[:, :K]
    parents, tokens = at // V, at % V
    scores = total.flatten(1).gather(1, at).float()
    return {"scores": scores, "parents": parents.int(), "tokens": tokens.int(), "finished": done.gather(1, parents) | (tokens == eos), "lengths": length.gather(1, parents)}


def _reorder(s):
    B, K = s["case"]["batch"], s["case"]["beams"]
    src = (s["parents"].long() + K * torch.arange(B, device=DEV)[:, None]).flatten()
    for t in s["states"]:
        t.copy_(t[src])
    return s["states"]


def run(state):
    s, kind = state, state["case"]["kind"]
    if kind == "append":
        if own:
            s["cache"].append(s["k"], s["v"], s["table"], s["positions"], s["rows"])
            k, v = s["cache"].read(s["table"], s["back"], s["back_rows"], tokens=s["total_back"], dtype=torch.bfloat16)
        else:
            k, v = _append(s)
        return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if kind == "attend":
        if own:
            c = s["case"]
            return s["cache"].attend(s["q"], s["table"], s["positions"], s["rows"], window=c["window"], keep_first=c["keep"], sink=c["sink"])
        return _attend(s)
    if kind == "select":
        if own:
            from moshi_amd.beam import beam_select
            r = beam_select(s["logits"], s["scores"], lengths=s["lengths"], finished=s["finished"], eos=2, length_penalty=s["case"]["penalty"])
            return {"scores": r.scores, "parents": r.parents, "tokens": r.tokens, "finished": r.finished, "lengths": r.lengths}
        return _select(s)
    if own:
        from moshi_amd.beam import beam_reorder
        beam_reorder(s["states"], s["parents"])
        return s["states"]
    return _reorder(s)


# --------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------------------------------
def work(case):
    if case["kind"] in ("append", "attend"):
        past, rows = _lengths(case)
        G, D, V, item = case["kv_heads"], case["dim"], case["vdim"], DTYPES[case["dtype"]].itemsize
        if case["kind"] == "append":
            new = sum(rows) * G * (D + V)
            held = sum(p % BLOCK + r for p, r in zip(past, rows)) * G * (D + V)            # tokens of the written blocks, read back
            return {"bytes": new * item + new + held + 2 * held, "flops": 8 * new}
        H, w = case["heads"], case["window"]
        keys = pairs = 0
        for p, r in zip(past, rows):
            seen = [min(p + i + 1, w + min(case["keep"], max(0, p + i + 1 - w))) if w else p + i + 1 for i in range(r)]
            pairs += sum(seen)
            keys += p + r if not w else min(p + r, w + r - 1 + case["keep"])
        return {"bytes": keys * G * (D + V) + keys * G // BLOCK * 8 + sum(rows) * H * (D + V) * item, "flops": 2 * pairs * H * (D + V)}
    B, K = case["batch"], case["beams"]
    if case["kind"] == "select":
        n = B * K * case["vocab"]
        return {"bytes": n * DTYPES[case["dtype"]].itemsize + 34 * B * K, "flops": 4 * n}
    row = case["layers"] * case["heads"] * (case["dim"] * case["vdim"] * DTYPES[case["dtype"]].itemsize + 12 * (2 * case["dim"] + case["vdim"])) + 4 * case["tokens"]
    return {"bytes": 2 * B * K * row, "flops": 0}


# --------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# --------------------------------------------------------------------------------------------------------------------
def _turn(x, pos, case):
    """Complex numbers times exp(i angle): x [heads, tokens, dim] in float64."""
    r = case["rot"]
    if not r:
        return x
    i = torch.arange(r // 2, device=x.device, dtype=torch.float64)
    turn = torch.polar(torch.ones((), device=x.device, dtype=torch.float64), pos.double()[:, None] * torch.exp(-2 * i / r * math.log(1e4)))
    at = torch.stack([i.long(), i.long() + r // 2] if case["halves"] else [2 * i.long(), 2 * i.long() + 1])
    z = torch.complex(x[..., at[0]], x[..., at[1]]) * turn
    y = x.clone()
    y[..., at[0]], y[..., at[1]] = z.real, z.imag
    return y


def _held(s, e, n, which):
    """Values of sequence e's first n tokens, [heads, n, dim] in float64."""
    pages = s["table"][e, :-(-n // PAGE)].long()
    codes, scale = s[which + "_codes"][pages].double(), s[which + "_scale"][pages].double()
    codes = codes.transpose(2, 3) if which == "v" else codes                               # [pages, heads, 64, dim]
    codes = codes.unflatten(2, (PAGE // BLOCK, BLOCK)) * scale[..., None, None]
    return codes.flatten(2, 3).transpose(0, 1).flatten(1, 2)[:, :n]


def _exact_append(case, s):
    past, rows = _lengths(case)
    top, out = TOP[case["codes"]], {"k": [], "v": []}
    scales = {"k_scale": s["k_scale"].double(), "v_scale": s["v_scale"].double()}
    row = 0
    for e, (p, r) in enumerate(zip(past, rows)):
        back = p // BLOCK * BLOCK
        for which in "kv":
            x = s[which][row:row + r].double().transpose(0, 1)                             # [heads, rows, dim]
            if which == "k":
                x = _turn(x, torch.arange(p, p + r, device=DEV), case)
            codes = s[which + "_codes"]
            parts = []
            for b in range(back, p + r, BLOCK):
                page, part = int(s["table"][e, b // PAGE]), b % PAGE // BLOCK
                lo, hi = max(b, p), min(b + BLOCK, p + r)
                scale = (x[:, lo - p:hi - p].abs().amax(dim=(1, 2)).clamp(min=TINY)) / top
                if lo > b:
                    before = s[which + "_scale"][page, :, part].double()
                    scale = torch.maximum(scale, before)
                    c = codes[page, :, :, b % PAGE:b % PAGE + lo - b].transpose(1, 2) if which == "v" else codes[page, :, b % PAGE:b % PAGE + lo - b]
                    parts.append(_to_code(c.double() * (before / scale)[:, None, None], case) * scale[:, None, None])
                parts.append(_to_code(x[:, lo - p:hi - p] / scale[:, None, None], case) * scale[:, None, None])
                scales[which + "_scale"][page, :, part] = scale
            out[which].append(torch.cat(parts, dim=1).transpose(0, 1))
        row += r
    return {"k": torch.cat(out["k"]), "v": torch.cat(out["v"]), **scales}


def _to_code(x, case):
    if case["codes"] == "int8":
        return x.round().clamp(-127, 127)
    # e4m3: 3 bits behind the leading one, the smallest step 2^-9
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return ((x / step).round() * step).clamp(-448, 448)


def _exact_attend(case, s):
    past, rows = _lengths(case)
    G, rep = case["kv_heads"], case["heads"] // case["kv_heads"]
    out, row = [], 0
    for e, (p, r) in enumerate(zip(past, rows)):
        n = p + r
        k, v = _held(s, e, n, "k"), _held(s, e, n, "v")
        pos = torch.arange(p, n, device=DEV)
        q = _turn(s["q"][row:row + r].double().transpose(0, 1), pos, case)
        got = []
        for h in range(case["heads"]):
            score = q[h] @ k[h // rep].T.contiguous() / math.sqrt(case["dim"])
            gap = pos[:, None] - torch.arange(n, device=DEV)
            seen = gap >= 0
            if case["window"]:
                seen &= (gap < case["window"]) | (torch.arange(n, device=DEV) < case["keep"])
            score[~seen] = -math.inf
            if case["sink"]:
                score = torch.cat([score, torch.zeros((r, 1), dtype=torch.float64, device=DEV)], dim=1)
            got.append(torch.softmax(score, dim=-1)[:, :n] @ v[h // rep])
        out.append(torch.stack(got, dim=1))
        row += r
    return torch.cat(out)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, s)
    if case["kind"] == "attend":
        return _exact_attend(case, s)
    B, K = case["batch"], case["beams"]
    if case["kind"] == "select":
        eos, best = 2, []
        logp = torch.log_softmax(s["logits"].double(), dim=-1).view(B, K, -1)
        for b in range(B):
            every = []
            for i in range(K):
                score, n = float(s["scores"][b, i]), int(s["lengths"][b, i])
                line = torch.full_like(logp[b, i], -math.inf) if s["finished"][b, i] else score + logp[b, i]
                if s["finished"][b, i]:
                    line[eos] = score
                every.append(torch.stack([line / float(n + (not s["finished"][b, i])) ** case["penalty"], line]))
            every = torch.cat(every, dim=1)
            best.append(every[1][torch.topk(every[0], K).indices])
        return {"scores": torch.stack(best), "parents": None, "tokens": None, "finished": None, "lengths": None}
    rows = [b * K + int(i) for b in range(B) for i in s["parents"][b]]
    return [torch.stack([t[i] for i in rows]) for t in s["states"]]
