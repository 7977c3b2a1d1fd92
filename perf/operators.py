"""The attention operators of a decode engine, and the cases that they are measured on.

  append   the new tokens' keys and values into a paged cache, the position rotation applied on the way, and the
           rotated queries (amdc.kv_append)
  decode   attention of one or a few new tokens per sequence over the paged cache (amdc.attn_decode)
  prefill  causal attention of whole prompts or prompt chunks of different lengths, packed (amdc.attn_prefill)

The cache is a pool of pages of `page` positions for every key / value head, in 16-bit floats, stored as the matrix
units read it:
  keys    [n_pages][n_kv][page / 16][hd / 8][16][8]: position 16 a + c, element 8 b + e at [a][b][c][e]
  values  [n_pages][n_kv][page / 8][hd][8]:          position 8 a + e, element d        at [a][d][e]
Sequence b's positions 0 .. len[b] - 1 (the new ones included) are in the pages pages[b][0], pages[b][1], ...
Rows of new tokens are packed: sequence b has the rows cu[b] .. cu[b + 1] - 1, or without cu T rows each.

Queries and outputs are 32-bit floats ("f32": the type of the library's GEMVs and GEMMs) or of the cache's type.

Where `own` is false, run() computes the operators in elementary torch operations; where it is true it calls the
library.
"""
import math
import os
import random
import sys

import torch

own = False

CACHE = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token of one sequence, 7B-class heads (32 of 128, no sharing): the latency of the call
        {"name": "append_1_7b", "op": "append", "type": "f16", "qtype": "f32", "n_q": 32, "n_kv": 32, "hd": 128, "page": 64, "rot": 128, "rope": "pairs",
         "seqs": 1, "lo": 700, "hi": 700, "new_lo": 1, "new_hi": 1},
        # a serving batch's step, 27B-class heads (24 over 4 of 256), a quarter of each head rotated
        {"name": "append_96_27b", "op": "append", "type": "bf16", "qtype": "bf16", "n_q": 24, "n_kv": 4, "hd": 256, "page": 32, "rot": 64, "rope": "halves",
         "seqs": 96, "lo": 40, "hi": 9000, "new_lo": 1, "new_hi": 1},
        # several prompts at once, the keys and values of a whole chunk each
        {"name": "append_prompts", "op": "append", "type": "f16", "qtype": "f16", "n_q": 32, "n_kv": 8, "hd": 128, "page": 16, "rot": 128, "rope": "halves",
         "seqs": 9, "lo": 150, "hi": 2600, "new_lo": 133, "new_hi": 2100},
        # batch-1 decode of a short chat, 7B-class heads: the smallest call, latency counts
        {"name": "decode_1_short_7b", "op": "decode", "type": "f16", "qtype": "f32", "n_q": 32, "n_kv": 32, "hd": 128, "page": 64, "T": 1, "window": 0,
         "seqs": 1, "lo": 421, "hi": 421},
        # batch-1 decode over a long document, 27B-class heads: few rows, split over the cache's length
        {"name": "decode_1_long_27b", "op": "decode", "type": "f16", "qtype": "f32", "n_q": 24, "n_kv": 4, "hd": 256, "page": 64, "T": 1, "window": 0,
         "seqs": 1, "lo": 60001, "hi": 60001},
        # a serving batch of chats of very different lengths, small pages
        {"name": "decode_64_ragged", "op": "decode", "type": "bf16", "qtype": "bf16", "n_q": 32, "n_kv": 8, "hd": 128, "page": 16, "T": 1, "window": 0,
         "seqs": 64, "lo": 30, "hi": 16000},
        # the verify step of speculative decoding: five tokens of every sequence
        {"name": "verify5_8_27b", "op": "decode", "type": "f16", "qtype": "f32", "n_q": 24, "n_kv": 4, "hd": 256, "page": 64, "T": 5, "window": 0,
         "seqs": 8, "lo": 900, "hi": 6000},
        # a single short prompt, 7B-class heads
        {"name": "prefill_77_7b", "op": "prefill", "type": "f16", "qtype": "f32", "n_q": 32, "n_kv": 32, "hd": 128, "page": 64, "window": 0,
         "seqs": 1, "lo": 77, "hi": 77, "new_lo": 77, "new_hi": 77},
        # the benchmark's prompt chunk of 256 tokens at the end of a longer prompt, 27B-class heads
        {"name": "prefill_chunk256_27b", "op": "prefill", "type": "f16", "qtype": "f32", "n_q": 24, "n_kv": 4, "hd": 256, "page": 64, "window": 0,
         "seqs": 1, "lo": 5000, "hi": 5000, "new_lo": 256, "new_hi": 256},
        # prompts of different lengths packed into one call, over a sliding window
        {"name": "prefill_packed_window", "op": "prefill", "type": "f16", "qtype": "f16", "n_q": 32, "n_kv": 8, "hd": 64, "page": 32, "window": 1024,
         "seqs": 11, "lo": 45, "hi": 2900, "new_lo": 45, "new_hi": 2900},
        # a long prompt at once, the largest call
        {"name": "prefill_long", "op": "prefill", "type": "bf16", "qtype": "bf16", "n_q": 32, "n_kv": 8, "hd": 128, "page": 64, "window": 0,
         "seqs": 1, "lo": 12000, "hi": 12000, "new_lo": 12000, "new_hi": 12000},
    ]


def _log(rng, lo, hi):
    return lo * (hi / lo) ** rng.random()


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prefill", "prefill"])
    n_q, n_kv, hd = rng.choice([(32, 32, 128), (32, 8, 128), (24, 4, 256), (32, 8, 64), (28, 4, 128), (16, 2, 256), (12, 12, 64)])
    ty = rng.choice(["f16", "bf16"])
    c = {"op": op, "type": ty, "qtype": rng.choice(["f32", ty]), "n_q": n_q, "n_kv": n_kv, "hd": hd, "page": rng.choice([16, 32, 64, 128])}
    if op == "append":
        decode = rng.random() < 0.5
        new_hi = 1 if decode else int(_log(rng, 2, 3000))
        new_lo = max(1, int(new_hi * rng.random()))
        seqs = max(1, min(int(_log(rng, 1, 200)), 12000 // new_hi))
        lo = new_hi + int(_log(rng, 1, 2000))
        return {**c, "rot": rng.choice([hd, hd // 2, hd // 4]), "rope": rng.choice(["pairs", "halves"]), "seqs": seqs, "lo": lo, "hi": lo + int(_log(rng, 1, 4000)),
                "new_lo": new_lo, "new_hi": new_hi}
    if op == "decode":
        # the cache read by one call stays under that of the largest listed one
        most = 500_000 * 1024 // (n_kv * hd)
        seqs = int(_log(rng, 1, 200))
        hi = max(20, min(int(_log(rng, 100, 100_000)), most // seqs))
        lo = max(9, int(hi * rng.random()))
        return {**c, "T": rng.choice([1, 1, 1, 2, 4, 8]), "window": rng.choice([0, 0, 0, int(_log(rng, 50, 4096))]), "seqs": seqs, "lo": lo, "hi": hi}
    # the scores of one call stay under those of the largest listed one
    seqs = rng.choice([1, 1, 2, 3, 5, 8, 16])
    new_hi = int(_log(rng, 17, 9000))
    hi = new_hi + rng.choice([0, 0, int(_log(rng, 10, 8000))])
    most = 32 * 11000 * 11000
    while seqs > 1 and seqs * new_hi * hi * n_q > most // 2:
        seqs -= 1
    while seqs * new_hi * hi * n_q * hd > most * 128:
        new_hi = new_hi * 4 // 5
        hi = max(new_hi, hi * 4 // 5)
    new_lo = max(1, int(new_hi * rng.random())) if seqs > 1 else new_hi
    return {**c, "window": rng.choice([0, 0, 0, int(_log(rng, 50, 4096))]), "seqs": seqs, "lo": hi if seqs == 1 else max(new_hi, hi - hi // 3), "hi": hi,
            "new_lo": new_lo, "new_hi": new_hi}


# ---------------------------------------------------------------- inputs

def _shape_of(case):
    """The sequences' lengths (new tokens included) and their numbers of new tokens: spread between the case's bounds, the
    same for every seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    n = case["seqs"]

    def spread(lo, hi):
        got = [min(hi, int(_log(rng, lo, hi + 1))) for _ in range(n)]
        got[rng.randrange(n)] = hi
        return got

    new = spread(case["new_lo"], case["new_hi"]) if "new_lo" in case else [case["T"]] * n
    if "new_lo" in case and case["lo"] == case["new_lo"] and case["hi"] == case["new_hi"]:
        return new, new  # whole prompts
    return [max(a, b) for a, b in zip(spread(case["lo"], case["hi"]), new)], new


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 13)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    length, new = _shape_of(case)
    n_q, n_kv, hd, page, n = case["n_q"], case["n_kv"], case["hd"], case["page"], case["seqs"]
    ty, qty = CACHE[case["type"]], CACHE.get(case["qtype"], torch.float32)
    held = [-(-v // page) for v in length]
    n_pages = sum(held) + 3
    # the pages of a pool in use: each sequence's are scattered over it; entries behind its last one are not read
    order = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros((n, max(held)), dtype=torch.int32)
    at = 0
    for b, k in enumerate(held):
        table[b, :k] = torch.arange(at, at + k)
        at += k
    used = torch.arange(max(held))[None, :] < torch.tensor(held)[:, None]
    pages = torch.where(used.cuda(), order[table.cuda().long()], torch.zeros((), dtype=torch.int32, device="cuda")).contiguous()
    rows = sum(new)
    cu = torch.tensor([sum(new[:b]) for b in range(n + 1)], dtype=torch.int32, device="cuda")
    s = {"case": case, "pages": pages, "len": torch.tensor(length, dtype=torch.int32, device="cuda"), "cu": cu, "rows": rows, "n_pages": n_pages, "most": max(length),
         "new_most": max(new)}
    s["k"] = randn(n_pages, n_kv, page // 16, hd // 8, 16, 8).to(ty)
    s["v"] = randn(n_pages, n_kv, page // 8, hd, 8).to(ty)
    if case["op"] == "append":
        # the fused projection's output rows: queries, keys, values side by side
        s["x"] = randn(rows, (n_q + 2 * n_kv) * hd)
        s["qo"] = torch.empty((rows, n_q * hd), dtype=qty, device="cuda")
        s["freq"] = (10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])).float().cuda()
    else:
        # scores with a deviation of about 2: a few positions carry most of a row's weight
        s["q"] = (2.0 * randn(rows, n_q * hd)).to(qty)
        s["y"] = torch.empty((rows, n_q * hd), dtype=qty, device="cuda")
    if own:
        amdc = _library()
        amdc.open_device()
        s["kv"] = amdc.Kv({"f16": amdc.TYPE_F16, "bf16": amdc.TYPE_BF16}[case["type"]], n_kv, hd, page, n_pages, s["k"].data_ptr(), s["v"].data_ptr(), n, pages.shape[1],
                          pages.data_ptr(), s["len"].data_ptr())
        s["qt"] = amdc.TYPE_F32 if qty == torch.float32 else s["kv"].type
        if case["op"] != "append":
            # the workspace of a serving loop: made once, cleared once
            size = amdc.attn_decode_ws(s["kv"], n_q, case["T"]) if case["op"] == "decode" else amdc.attn_prefill_ws(s["kv"], n_q, rows)
            s["ws"] = torch.zeros((size,), dtype=torch.uint8, device="cuda")
    return s


def _library():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "amd.c_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import amdc
    return amdc


# ---------------------------------------------------------------- one pass

def run(s):
    return _calls(s) if own else _plain(s)


def _calls(s):
    amdc, case = _library(), s["case"]
    n_q, n_kv, hd = case["n_q"], case["n_kv"], case["hd"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "append":
        x, w = s["x"].data_ptr(), (n_q + 2 * n_kv) * hd
        decode = case["new_hi"] == 1
        amdc.kv_append(s["kv"], x + 4 * n_q * hd, x + 4 * (n_q + n_kv) * hd, x, s["qo"].data_ptr(), s["qt"], n_q, 1 if decode else s["rows"], ks=w, vs=w, qs=w, qos=n_q * hd,
                       cu=None if decode else s["cu"].data_ptr(), freq=s["freq"].data_ptr(), n_rot=case["rot"],
                       rope=amdc.ROPE_PAIRS if case["rope"] == "pairs" else amdc.ROPE_HALVES, stream=stream)
        return {"k": s["k"], "v": s["v"], "q": s["qo"]}
    if case["op"] == "decode":
        amdc.attn_decode(s["kv"], s["q"].data_ptr(), s["y"].data_ptr(), s["qt"], n_q, case["T"], n_q * hd, n_q * hd, 1.0 / math.sqrt(hd), s["ws"].data_ptr(), s["ws"].numel(),
                         window=case["window"], stream=stream)
    else:
        amdc.attn_prefill(s["kv"], s["q"].data_ptr(), s["y"].data_ptr(), s["qt"], n_q, s["rows"], n_q * hd, n_q * hd, 1.0 / math.sqrt(hd), s["ws"].data_ptr(), s["ws"].numel(),
                          cu=s["cu"].data_ptr(), window=case["window"], stream=stream)
    return s["y"]


def _plain(s):
    case = s["case"]
    n_q, n_kv, hd, page, n = case["n_q"], case["n_kv"], case["hd"], case["page"], case["seqs"]
    cu, length = s["cu"].long(), s["len"].long()
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(cu[1:], row, right=True)
    pos = length[seq] - (cu[seq + 1] - cu[seq]) + row - cu[seq]
    if case["op"] == "append":
        q, k, v = s["x"].split([n_q * hd, n_kv * hd, n_kv * hd], 1)
        angle = pos[:, None].double() * s["freq"].double()
        cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]

        def rotated(x, heads):
            x = x.reshape(s["rows"], heads, hd)
            r, rest = x[..., :case["rot"]], x[..., case["rot"]:]
            a, b = (r[..., 0::2], r[..., 1::2]) if case["rope"] == "pairs" else r.chunk(2, -1)
            a, b = a * cos - b * sin, a * sin + b * cos
            r = torch.stack([a, b], -1).flatten(-2) if case["rope"] == "pairs" else torch.cat([a, b], -1)
            return torch.cat([r, rest], -1)

        slot, at = pos % page, s["pages"].long()[seq, pos // page]
        s["k"][at, :, slot // 16, :, slot % 16, :] = rotated(k, n_kv).reshape(s["rows"], n_kv, hd // 8, 8).to(s["k"].dtype)
        s["v"][at, :, slot // 8, :, slot % 8] = v.reshape(s["rows"], n_kv, hd).to(s["v"].dtype)
        s["qo"].copy_(rotated(q, n_q).flatten(1))
        return {"k": s["k"], "v": s["v"], "q": s["qo"]}
    # the cache of every sequence, [n][n_kv][positions][hd], and its queries, padded to the longest's number of rows
    table = s["pages"].long()
    k = s["k"][table].permute(0, 2, 1, 3, 5, 4, 6).reshape(n, n_kv, -1, hd)[:, :, :s["most"]].float().contiguous()
    v = s["v"][table].permute(0, 2, 1, 3, 5, 4).reshape(n, n_kv, -1, hd)[:, :, :s["most"]].float().contiguous()
    t, group = s["new_most"], n_q // n_kv
    inner = row - cu[seq]
    q = torch.zeros((n, t, n_q * hd), device="cuda")
    q[seq, inner] = s["q"].float()
    q = q.view(n, t, n_kv, group, hd).permute(0, 2, 3, 1, 4).reshape(n, n_kv, group * t, hd)
    at = torch.full((n, t), -1, device="cuda")
    at[seq, inner] = pos
    j = torch.arange(s["most"], device="cuda")
    seen = j <= at[:, :, None]
    if case["window"]:
        seen &= j > at[:, :, None] - case["window"]
    seen = seen[:, None, None]
    score = torch.matmul(q, k.transpose(2, 3)).mul_(1.0 / math.sqrt(hd)).view(n, n_kv, group, t, -1).masked_fill_(~seen, -math.inf)
    score -= score.amax(-1, keepdim=True).clamp_min_(-3e38)
    p = score.exp_()
    total = p.sum(-1, keepdim=True).clamp_min_(1e-30)
    y = torch.matmul(p.view(n, n_kv, group * t, -1), v).view(n, n_kv, group, t, hd) / total
    s["y"].copy_(y.permute(0, 3, 1, 2, 4).reshape(n, t, n_q * hd)[seq, inner])
    return s["y"]


# ---------------------------------------------------------------- what a pass cannot do without, and its result in 64 bits

def work(case):
    length, new = _shape_of(case)
    n_q, n_kv, hd = case["n_q"], case["n_kv"], case["hd"]
    rows, qb = sum(new), 4 if case["qtype"] == "f32" else 2
    tables = 4 * sum(-(-v // case["page"]) for v in length) + 8 * len(length)
    if case["op"] == "append":
        return {"bytes": rows * hd * ((n_q + 2 * n_kv) * 4 + n_q * qb + n_kv * 4) + tables, "flops": 3 * rows * (n_q + n_kv) * case["rot"]}
    w = case["window"] or max(length)
    pairs = sum(min(p + 1, w) for a, m in zip(length, new) for p in range(a - m, a))
    read = sum(a - max(0, a - m + 1 - w) for a, m in zip(length, new))
    return {"bytes": read * n_kv * hd * 4 + 2 * rows * n_q * hd * qb + tables, "flops": 4 * pairs * n_q * hd}


def exact(case, seed):
    s = prepare(case, seed)
    length, new = _shape_of(case)
    n_q, n_kv, hd, page, G = case["n_q"], case["n_kv"], case["hd"], case["page"], case["n_q"] // case["n_kv"]
    pages = s["pages"].cpu().tolist()
    if case["op"] == "append":
        K, V, Q = s["k"].double(), s["v"].double(), torch.empty((s["rows"], n_q * hd), dtype=torch.float64, device="cuda")
        first = 0
        for b in range(case["seqs"]):
            m = new[b]
            x = s["x"][first:first + m].double().view(m, n_q + 2 * n_kv, hd)
            where = torch.arange(length[b] - m, length[b], device="cuda")
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), where[:, None].double() * s["freq"].double()[None, :])[:, None, :]
            half = case["rot"] // 2
            i = torch.arange(half, device="cuda")
            lo, hi = (2 * i, 2 * i + 1) if case["rope"] == "pairs" else (i, i + half)
            r = x.clone()
            z = torch.complex(x[:, :n_q + n_kv, lo], x[:, :n_q + n_kv, hi]) * turn
            r[:, :n_q + n_kv, lo], r[:, :n_q + n_kv, hi] = z.real, z.imag
            Q[first:first + m] = r[:, :n_q].reshape(m, -1)
            page_of = torch.tensor(pages[b], device="cuda")[where // page]
            inside = where % page
            for h in range(n_kv):
                K[page_of, h, inside // 16, :, inside % 16] = r[:, n_q + h].view(m, hd // 8, 8)
                V[page_of, h, inside // 8, :, inside % 8] = x[:, n_q + n_kv + h]
            first += m
        return {"k": K, "v": V, "q": Q}
    Y = torch.empty((s["rows"], n_q, hd), dtype=torch.float64, device="cuda")
    scale, first = 1.0 / math.sqrt(hd), 0
    for b in range(case["seqs"]):
        L, m = length[b], new[b]
        held = torch.tensor(pages[b][:-(-L // page)], device="cuda")
        begin = max(0, L - m + 1 - case["window"]) if case["window"] else 0
        j = torch.arange(begin, L, device="cuda")
        i = torch.arange(L - m, L, device="cuda")[:, None]
        hidden = j > i
        if case["window"]:
            hidden = hidden | (i - j >= case["window"])
        for h in range(n_kv):
            k = s["k"][held, h].transpose(2, 3).reshape(-1, hd)[begin:L].double()
            v = s["v"][held, h].transpose(2, 3).reshape(-1, hd)[begin:L].double()
            for u in range(G):
                q = s["q"][first:first + m].view(m, n_q, hd)[:, h * G + u].double()
                e = (q @ k.t() * scale).masked_fill(hidden, -math.inf)
                Y[first:first + m, h * G + u] = torch.softmax(e, 1) @ v
        first += m
    return Y.view(s["rows"], n_q * hd)
