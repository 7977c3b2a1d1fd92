"""The operators of a linear-attention layer of a decode engine, and the cases that they are measured on.

  conv     the short causal convolution over the layer's input channels, with its state (amdc.conv)
  decode   the gated delta rule, one or a few new tokens of every sequence (amdc.gdn_decode)
  prefill  the gated delta rule over whole prompts or prompt chunks of different lengths, packed (amdc.gdn_prefill)
  gate     the norm of the layer's heads, times their gate (amdc.norm_gate_q8)
  res      the norm behind a block, the scaled residual, and the norm before the next block (amdc.norm_res_q8)

A sequence's state of the delta rule is, for every value head, a matrix S of dk x dv floats; for a token with the row
vectors q, k, v, decay exp(g) and rate beta of that head

  S <- exp(g) S,   u = beta (v - k S),   S <- S + k^T u,   y = q S

with k / sqrt(k.k + eps) for k, scale q / sqrt(q.q + eps) for q, g = A softplus(a + dt) and beta = sigmoid(b). States are
kept in slots of a pool, [n_slots][n_v][dv / 16][dk][16]: row i, column 16 a + c at [a][i][c]. A sequence starts from
slot from[b] (-1: a state of zeros) and leaves its new state in slot to[b] (-1: nowhere); a verify step leaves one after
every token. The convolution's state is the last width - 1 inputs, [n_slots][width - 1][channels].

Where `own` is false, run() computes the operators in elementary torch operations; where it is true it calls the
library.
"""
import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CHUNK = 64


def listed():
    big = {"n_k": 16, "n_v": 48, "dk": 128, "dv": 128, "order": "tiled"}
    return [
        # one token of one sequence, 27B-class layer (16 heads of keys, 48 of values, 128 each): the latency of the call
        {"name": "conv_1_27b", "op": "conv", "type": "f32", "ch": 10240, "width": 4, "seqs": 1, "new_lo": 1, "new_hi": 1, "each": False},
        # several prompts at once, some of them continued
        {"name": "conv_prompts", "op": "conv", "type": "bf16", "ch": 8192, "width": 4, "seqs": 9, "new_lo": 133, "new_hi": 2100, "each": False},
        # batch-1 decode: the smallest call, latency counts
        {"name": "decode_1_27b", "op": "decode", "type": "f32", **big, "T": 1, "seqs": 1, "each": False},
        # a serving batch's step, every state read and written once
        {"name": "decode_96", "op": "decode", "type": "bf16", "n_k": 16, "n_v": 32, "dk": 128, "dv": 128, "order": "grouped", "T": 1, "seqs": 96, "each": False},
        # the verify step of speculative decoding: five tokens of every sequence, the state kept after each
        {"name": "verify5_8_27b", "op": "decode", "type": "f32", **big, "T": 5, "seqs": 8, "each": True},
        # a single short prompt
        {"name": "prefill_77_27b", "op": "prefill", "type": "f32", **big, "seqs": 1, "new_lo": 77, "new_hi": 77, "fresh": 1.0},
        # prompts and chunks of prompts of different lengths packed into one call, heads of 64
        {"name": "prefill_packed", "op": "prefill", "type": "f16", "n_k": 8, "n_v": 16, "dk": 64, "dv": 64, "order": "grouped", "seqs": 11, "new_lo": 45, "new_hi": 2900,
         "fresh": 0.5},
        # a long prompt at once, the largest call
        {"name": "prefill_long_27b", "op": "prefill", "type": "f32", **big, "seqs": 1, "new_lo": 12000, "new_hi": 12000, "fresh": 1.0},
        # one token's heads before the output matrix
        {"name": "gate_1_27b", "op": "gate", "type": "f32", "n_h": 48, "hd": 128, "rows": 1, "gate": "silu"},
        # a prompt's
        {"name": "gate_4097", "op": "gate", "type": "bf16", "n_h": 32, "hd": 128, "rows": 4097, "gate": "silu"},
        # one token between two blocks, normed behind the first
        {"name": "res_1_27b", "op": "res", "n": 5120, "rows": 1, "post": True, "scale": 1.0},
        # a prompt between two blocks, its residual scaled
        {"name": "res_3001", "op": "res", "n": 4096, "rows": 3001, "post": True, "scale": 0.22},
    ]


def _log(rng, lo, hi):
    return lo * (hi / lo) ** rng.random()


def draw(rng):
    op = rng.choice(["conv", "decode", "decode", "prefill", "prefill", "gate", "res"])
    ty = rng.choice(["f32", "f16", "bf16"])
    if op == "gate":
        n_h, hd = rng.choice([(48, 128), (32, 128), (16, 256), (24, 64), (5, 128), (12, 32)])
        return {"op": op, "type": ty, "n_h": n_h, "hd": hd, "rows": int(_log(rng, 1, 8000)), "gate": rng.choice(["silu", "sigmoid"])}
    if op == "res":
        return {"op": op, "n": 32 * int(_log(rng, 8, 400)), "rows": int(_log(rng, 1, 5000)), "post": rng.random() < 0.7, "scale": rng.choice([1.0, 0.22, 0.7])}
    if op == "conv":
        decode = rng.random() < 0.5
        new_hi = rng.choice([1, 1, 2, 5, 8]) if decode else int(_log(rng, 9, 4000))
        seqs = max(1, min(int(_log(rng, 1, 200)), 12000 // new_hi))
        return {"op": op, "type": ty, "ch": rng.choice([10240, 8192, 4096, 2050, 1001, 3 * int(_log(rng, 20, 2000))]), "width": rng.choice([4, 4, 4, 3, 2]), "seqs": seqs,
                "new_lo": new_hi if decode else max(1, int(new_hi * rng.random())), "new_hi": new_hi, "each": decode and new_hi > 1}
    n_k, n_v = rng.choice([(16, 48), (16, 32), (16, 16), (8, 16), (4, 4), (2, 10), (1, 3), (6, 6)])
    dk, dv = rng.choice([(128, 128), (128, 128), (64, 64), (64, 128), (128, 64), (128, 256), (64, 48)])
    c = {"op": op, "type": ty, "n_k": n_k, "n_v": n_v, "dk": dk, "dv": dv, "order": rng.choice(["tiled", "grouped"])}
    if op == "decode":
        T = rng.choice([1, 1, 1, 2, 4, 8])
        # the states written by one call stay under 500 MB
        seqs = max(1, min(int(_log(rng, 1, 300)), 500_000_000 // (n_v * dk * dv * 4 * T)))
        return {**c, "T": T, "seqs": seqs, "each": T > 1 and rng.random() < 0.8}
    seqs = rng.choice([1, 1, 2, 3, 5, 8, 16])
    new_hi = int(_log(rng, 2, 9000))
    # the tokens times heads of one call, padded to the longest, stay under the largest listed one's
    while seqs > 1 and seqs * new_hi > 20000:
        seqs -= 1
    while seqs * new_hi * n_v * dk * dv > 12000 * 48 * 128 * 128:
        new_hi = new_hi * 4 // 5
    new_lo = max(1, int(new_hi * rng.random())) if seqs > 1 else new_hi
    return {**c, "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi, "fresh": rng.choice([0.0, 0.5, 1.0])}


# ---------------------------------------------------------------- inputs

def _new(case):
    """The sequences' numbers of new tokens: spread between the case's bounds, the same for every seed."""
    if "T" in case:
        return [case["T"]] * case["seqs"]
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    lo, hi, n = case["new_lo"], case["new_hi"], case["seqs"]
    got = [min(hi, int(_log(rng, lo, hi + 1))) for _ in range(n)]
    got[rng.randrange(n)] = hi
    return got


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 7919 + 13)
    return g


def prepare(case, seed):
    g = _generator(seed)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=g)

    s = {"case": case}
    if own:
        _library().open_device()
    if case["op"] == "gate":
        rows, w = case["rows"], case["n_h"] * case["hd"]
        s["x"], s["z"] = (0.3 * randn(rows, w)).to(TYPES[case["type"]]), randn(rows, w)
        s["w"], s["y"] = 1 + 0.1 * randn(case["hd"]), torch.empty((rows, w), device="cuda")
        return s
    if case["op"] == "res":
        rows, n = case["rows"], case["n"]
        s["x"], s["res"] = 3 * randn(rows, n), 20 * randn(rows, n)
        s["w1"], s["w2"] = 1 + 0.1 * randn(n), 1 + 0.1 * randn(n)
        s["h"], s["y"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        return s
    new = _new(case)
    n, rows = len(new), sum(new)
    s["rows"], s["new"] = rows, new
    s["cu"] = torch.tensor([sum(new[:b]) for b in range(n + 1)], dtype=torch.int32, device="cuda")
    each = case.get("each", False)
    kept = rows if each else n
    # the slots of a pool in use: decode in place, a verify step and a prompt into others; prompts that begin have none to start from
    verify, begins = each or case["op"] == "prefill", case["op"] == "prefill" or (case["op"] == "conv" and case["new_hi"] > 8)
    n_slots = n + (kept if verify else 0) + 3
    order = torch.randperm(n_slots, device="cuda", generator=g).to(torch.int32)
    s["to"] = order[n:n + kept].contiguous() if verify else order[:n].contiguous()
    s["from"] = order[:n].clone()
    if begins:
        s["from"][torch.rand(n, device="cuda", generator=g) < case.get("fresh", 0.5)] = -1
    s["n_slots"], s["each"] = n_slots, each
    ty = TYPES[case["type"]]
    if case["op"] == "conv":
        ch, wd = case["ch"], case["width"]
        s["state"], s["x"] = randn(n_slots, wd - 1, ch), randn(rows, ch)
        s["w"], s["bias"] = randn(ch, wd) / math.sqrt(wd), 0.1 * randn(ch)
        s["y"] = torch.empty((rows, ch), dtype=ty, device="cuda")
    else:
        n_k, n_v, dk, dv = case["n_k"], case["n_v"], case["dk"], case["dv"]
        s["state"] = 0.3 * randn(n_slots, n_v, dv // 16, dk, 16)
        # the convolution's output rows: queries, keys, values side by side, each a SiLU of something normal
        x = randn(rows, 2 * n_k * dk + n_v * dv)
        s["x"] = (x * torch.sigmoid(x)).to(ty)
        # decays of 0.2 to 0.999 a token at a = 0
        s["A"] = -torch.exp(torch.rand(n_v, device="cuda", generator=g) * math.log(16.0))
        dt = 0.001 * 100.0 ** torch.rand(n_v, device="cuda", generator=g)
        s["dt"] = torch.log(torch.expm1(dt))
        s["ab"] = randn(rows, 2 * n_v)
        s["y"] = torch.empty((rows, n_v * dv), dtype=ty, device="cuda")
    if own:
        amdc = _library()
        s["slots"] = amdc.Slots(n, n_slots, s["from"].data_ptr(), s["to"].data_ptr())
        s["t"] = {"f32": amdc.TYPE_F32, "f16": amdc.TYPE_F16, "bf16": amdc.TYPE_BF16}[case["type"]]
        if case["op"] != "conv":
            s["gdn"] = amdc.Gdn(n_k, n_v, dk, dv, amdc.HEADS_TILED if case["order"] == "tiled" else amdc.HEADS_GROUPED, 1.0 / math.sqrt(dk), 1e-6, s["A"].data_ptr(),
                                s["dt"].data_ptr())
        if case["op"] == "prefill":
            # the workspace of a serving loop
            s["ws"] = torch.zeros((amdc.gdn_prefill_ws(s["gdn"], n, rows),), dtype=torch.uint8, device="cuda")
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
    stream = torch.cuda.current_stream().cuda_stream
    op, y = case["op"], s["y"].data_ptr()
    if op == "gate":
        n_h, hd = case["n_h"], case["hd"]
        t = {"f32": amdc.TYPE_F32, "f16": amdc.TYPE_F16, "bf16": amdc.TYPE_BF16}[case["type"]]
        w = n_h * hd
        amdc.norm_gate_q8(s["x"].data_ptr(), t, s["w"].data_ptr(), s["z"].data_ptr(), y, n_h, hd, 1e-6, amdc.GATE_SILU if case["gate"] == "silu" else amdc.GATE_SIGMOID,
                          T=case["rows"], xs=w * s["x"].element_size(), zs=4 * w, ys=4 * w, stream=stream)
        return s["y"]
    if op == "res":
        n = case["n"]
        amdc.norm_res_q8(s["x"].data_ptr(), s["w1"].data_ptr() if case["post"] else None, case["scale"], s["res"].data_ptr(), s["h"].data_ptr(), s["w2"].data_ptr(), y, n, 1e-6,
                         T=case["rows"], xs=4 * n, rs=4 * n, hs=4 * n, ys=4 * n, stream=stream)
        return {"h": s["h"], "y": s["y"]}
    T = case["T"] if op == "decode" else case["new_hi"] if op == "conv" and (s["each"] or case["new_hi"] == 1) else None
    if op == "conv":
        ch = case["ch"]
        amdc.conv(s["slots"], s["state"].data_ptr(), s["x"].data_ptr(), s["w"].data_ptr(), s["bias"].data_ptr(), y, s["t"], ch, case["width"], T or s["rows"], ch, ch,
                  cu=None if T else s["cu"].data_ptr(), each=s["each"], act=amdc.ACT_SILU, stream=stream)
        return {"y": s["y"], "state": s["state"]}
    n_k, n_v, dk, dv = case["n_k"], case["n_v"], case["dk"], case["dv"]
    q, xs, es = s["x"].data_ptr(), s["x"].shape[1], s["x"].element_size()
    k, v, a = q + es * n_k * dk, q + es * 2 * n_k * dk, s["ab"].data_ptr()
    if op == "decode":
        amdc.gdn_decode(s["gdn"], s["slots"], s["state"].data_ptr(), q, k, v, a, a + 4 * n_v, y, s["t"], T, xs, xs, xs, 2 * n_v, 2 * n_v, n_v * dv, each=s["each"], stream=stream)
    else:
        amdc.gdn_prefill(s["gdn"], s["slots"], s["state"].data_ptr(), q, k, v, a, a + 4 * n_v, y, s["t"], s["rows"], xs, xs, xs, 2 * n_v, 2 * n_v, n_v * dv, s["ws"].data_ptr(),
                         s["ws"].numel(), cu=s["cu"].data_ptr(), stream=stream)
    return {"y": s["y"], "state": s["state"]}


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "gate":
        x = s["x"].float().view(case["rows"], case["n_h"], case["hd"])
        z = s["z"].view_as(x)
        x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * s["w"]
        g = 1.0 / (1.0 + torch.exp(-z))
        s["y"].copy_((x * (z * g if case["gate"] == "silu" else g)).flatten(1))
        return s["y"]
    if op == "res":
        x = s["x"]
        if case["post"]:
            x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * s["w1"]
        h = s["res"] + case["scale"] * x
        s["h"].copy_(h)
        s["y"].copy_(h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * s["w2"])
        return {"h": s["h"], "y": s["y"]}
    # the rows' sequences and places in them; a sequence without a slot starts from zeros
    cu, new, n, each = s["cu"].long(), s["new"], len(s["new"]), s["each"]
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(cu[1:], row, right=True)
    at = row - cu[seq]
    most = max(new)
    start, to = s["from"].long(), s["to"].long()
    begin = torch.where((start >= 0).view(-1, *[1] * (s["state"].dim() - 1)), s["state"][start.clamp_min(0)], torch.zeros((), device="cuda"))
    if op == "conv":
        wd = case["width"]
        x = torch.zeros((n, wd - 1 + most, case["ch"]), device="cuda")
        x[:, :wd - 1] = begin
        x[seq, wd - 1 + at] = s["x"]
        y = s["bias"].expand(s["rows"], -1)
        for j in range(wd):
            y = y + s["w"][:, j] * x[seq, at + j]
        s["y"].copy_(y / (1.0 + torch.exp(-y)))
        b, last = (seq, at + 1) if each else (torch.arange(n, device="cuda"), cu[1:] - cu[:-1])
        s["state"][to] = x[b[:, None], last[:, None] + torch.arange(wd - 1, device="cuda")]
        return {"y": s["y"], "state": s["state"]}
    n_k, n_v, dk, dv = case["n_k"], case["n_v"], case["dk"], case["dv"]
    head = torch.arange(n_v, device="cuda")
    head = head % n_k if case["order"] == "tiled" else head // (n_v // n_k)
    q, k, v = s["x"].float().split([n_k * dk, n_k * dk, n_v * dv], 1)
    q, k, v = q.reshape(-1, n_k, dk), k.reshape(-1, n_k, dk), v.reshape(-1, n_v, dv)
    q = q * (q.square().sum(-1, keepdim=True) + 1e-6).rsqrt() * (1.0 / math.sqrt(dk))
    k = k * (k.square().sum(-1, keepdim=True) + 1e-6).rsqrt()
    a, b = s["ab"].split([n_v, n_v], 1)
    a = a + s["dt"]
    decay = s["A"] * (a.clamp_min(0) + torch.log1p(torch.exp(-a.abs())))
    rate = 1.0 / (1.0 + torch.exp(-b))
    S = begin.permute(0, 1, 3, 2, 4).reshape(n, n_v, dk, dv)

    def slot(S):
        return S.view(-1, n_v, dk, dv // 16, 16).transpose(2, 3)

    if op == "decode":
        T = case["T"]
        q, k, v = (t.reshape(n, T, -1, t.shape[-1]) for t in (q[:, head], k[:, head], v))
        decay, rate = decay.exp().view(n, T, n_v, 1, 1), rate.view(n, T, n_v, 1)
        y, kept = [], []
        for t in range(T):  # each token's state follows from the last one's
            S = S * decay[:, t]
            u = rate[:, t] * (v[:, t] - (k[:, t, :, :, None] * S).sum(-2))
            S = S + k[:, t, :, :, None] * u[:, :, None, :]
            y.append((q[:, t, :, :, None] * S).sum(-2))
            kept.append(S)
        s["y"].copy_(torch.stack(y, 1).reshape(n * T, -1))
        s["state"][to] = slot(torch.stack(kept, 1).flatten(0, 1)) if each else slot(S)
        return {"y": s["y"], "state": s["state"]}
    # chunks of 64 tokens: inside one, the tokens' updates solve a triangular system; from one to the next goes the state
    nc = -(-most // CHUNK)

    def chunks(x, heads):
        got = torch.zeros((n, nc * CHUNK, heads) + x.shape[2:], dtype=x.dtype, device="cuda")
        got[seq, at] = x
        return got.view(n, nc, CHUNK, heads, -1).transpose(2, 3).contiguous()

    q, k, v, rate = chunks(q, n_k), chunks(k, n_k), chunks(v, n_v), chunks(rate[:, :, None], n_v)
    G = chunks(decay.double()[:, :, None], n_v).cumsum(-2)  # in 64 bits: differences of it count
    kk, qk = (torch.matmul(x, k.transpose(-1, -2).contiguous())[:, :, head] for x in (k, q))
    lower = torch.ones((CHUNK, CHUNK), dtype=torch.bool, device="cuda").tril()
    D = (G - G.transpose(-1, -2)).masked_fill(~lower, -math.inf).exp().float()
    L = (rate * kk * D).tril(-1)
    M = torch.eye(CHUNK, device="cuda").expand(L.shape).contiguous()
    for i in range(1, CHUNK):  # a row of the inverse from those above it, all chunks at once
        M[..., i, :i] = -torch.matmul(L[..., i:i + 1, :i], M[..., :i, :i])[..., 0, :]
    qk = qk * D
    since, until, whole = G.exp().float(), (G[..., -1:, :] - G).exp().float(), G[..., -1:, :].exp().float()
    q, k = q[:, :, head], k[:, :, head]
    U, W = torch.matmul(M, rate * v), torch.matmul(M, rate * since * k)
    q, k = q * since, (k * until).transpose(-1, -2).contiguous()
    y = torch.empty((n, nc, n_v, CHUNK, dv), device="cuda")
    for c in range(nc):  # a chunk's state follows from the last one's
        new_v = U[:, c] - torch.matmul(W[:, c], S)
        y[:, c] = torch.matmul(q[:, c], S) + torch.matmul(qk[:, c], new_v)
        S = whole[:, c] * S + torch.matmul(k[:, c], new_v)
    s["y"].copy_(y.transpose(2, 3).reshape(n, nc * CHUNK, -1)[seq, at])
    s["state"][to] = slot(S)
    return {"y": s["y"], "state": s["state"]}


# ---------------------------------------------------------------- what a pass cannot do without, and its result in 64 bits

def work(case):
    eb = 4 if case.get("type") == "f32" else 2
    if case["op"] == "gate":
        n = case["rows"] * case["n_h"] * case["hd"]
        return {"bytes": n * (eb + 8) + 4 * case["hd"], "flops": 8 * n}
    if case["op"] == "res":
        n = case["rows"] * case["n"]
        return {"bytes": 16 * n + 8 * case["n"], "flops": 9 * n}
    new = _new(case)
    n, rows = len(new), sum(new)
    kept = rows if case.get("each") else n
    started = n * (1.0 - case.get("fresh", 0.5)) if case["op"] == "prefill" or (case["op"] == "conv" and case["new_hi"] > 8) else n
    if case["op"] == "conv":
        ch, wd = case["ch"], case["width"]
        return {"bytes": int(rows * ch * (4 + eb) + 4 * ch * (wd - 1) * (started + kept) + 4 * ch * (wd + 1)), "flops": rows * ch * (2 * wd + 4)}
    n_k, n_v, dk, dv = case["n_k"], case["n_v"], case["dk"], case["dv"]
    state = 4 * n_v * dk * dv
    return {"bytes": int(rows * (eb * (2 * n_k * dk + 2 * n_v * dv) + 8 * n_v) + state * (started + kept) + 8 * n_v), "flops": 7 * rows * n_v * dk * dv}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gate":
        x, z = s["x"].double().unflatten(1, (case["n_h"], case["hd"])), s["z"].double().unflatten(1, (case["n_h"], case["hd"]))
        y = x / torch.sqrt((x * x).mean(2, True) + 1e-6) * s["w"].double() * torch.sigmoid(z)
        return (y * z if case["gate"] == "silu" else y).flatten(1)
    if case["op"] == "res":
        def norm(x, w):
            return x / torch.sqrt((x * x).mean(1, True) + 1e-6) * w.double()
        x = s["x"].double()
        h = s["res"].double() + case["scale"] * (norm(x, s["w1"]) if case["post"] else x)
        return {"h": h, "y": norm(h, s["w2"])}
    new, each = s["new"], s["each"]
    state = s["state"].double()
    start, to, first = s["from"].tolist(), s["to"].tolist(), [sum(new[:b]) for b in range(len(new))]
    old = state.clone()
    if case["op"] == "conv":
        wd = case["width"]
        w, ys = s["w"].double(), []
        for b, m in enumerate(new):
            x = s["x"][first[b]:first[b] + m].double()
            x = torch.cat([old[start[b]] if start[b] >= 0 else torch.zeros_like(old[0]), x])
            windows = x.unfold(0, wd, 1)  # [m][ch][wd]
            y = (windows * w).sum(-1) + s["bias"].double()
            ys.append(y * torch.sigmoid(y))
            for t in range(m) if each else (m - 1,):
                state[to[first[b] + t if each else b]] = x[t + 1:t + wd]
        return {"y": torch.cat(ys), "state": state}
    n_k, n_v, dk, dv = case["n_k"], case["n_v"], case["dk"], case["dv"]
    head = [h % n_k if case["order"] == "tiled" else h * n_k // n_v for h in range(n_v)]
    x = s["x"].double()
    q = x[:, :n_k * dk].unflatten(1, (n_k, dk))
    k = x[:, n_k * dk:2 * n_k * dk].unflatten(1, (n_k, dk))
    v = x[:, 2 * n_k * dk:].unflatten(1, (n_v, dv))
    q = (q / torch.sqrt((q * q).sum(2, True) + 1e-6) / math.sqrt(dk))[:, head]
    k = (k / torch.sqrt((k * k).sum(2, True) + 1e-6))[:, head]
    ab = s["ab"].double()
    decay = torch.exp(s["A"].double() * torch.nn.functional.softplus(ab[:, :n_v] + s["dt"].double(), threshold=60.0))
    rate = torch.sigmoid(ab[:, n_v:])
    ys = torch.empty((s["rows"], n_v, dv), dtype=torch.float64, device="cuda")
    # token after token; sequences side by side, the longest first, so that those that still run are the first ones
    by = sorted(range(len(new)), key=lambda b: -new[b])
    S = torch.stack([old[start[b]].transpose(1, 2).reshape(n_v, dk, dv) if start[b] >= 0 else torch.zeros((n_v, dk, dv), dtype=torch.float64, device="cuda") for b in by])
    base = torch.tensor([first[b] for b in by], device="cuda")
    for t in range(max(new)):
        m = sum(new[b] > t for b in by)
        r, live = base[:m] + t, S[:m]
        live *= decay[r][:, :, None, None]
        u = rate[r][:, :, None] * (v[r] - torch.matmul(k[r][:, :, None, :], live)[:, :, 0])
        live += k[r][:, :, :, None] * u[:, :, None, :]
        ys[r] = torch.matmul(q[r][:, :, None, :], live)[:, :, 0]
        for i in range(m):
            if each or new[by[i]] == t + 1:
                state[to[first[by[i]] + t if each else by[i]]] = live[i].unflatten(2, (dv // 16, 16)).transpose(1, 2)
    return {"y": ys.flatten(1), "state": state}
