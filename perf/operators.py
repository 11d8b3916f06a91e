"""What the paged key-value cache and its attention are measured on.

Four operators of ``moss_tts._runtime.kernels``, as a server of ragged requests uses them one after the
other: ``qk_rope_paged`` (head norm, rotary position, new key and value rows into the pages),
``paged_attention_prompt`` and ``packed_attention`` (causal attention of packed prompts, over the pages
or over packed keys and values) and ``paged_attention_decode`` (one new token per sequence).

``run`` calls them where ``own`` is true and computes the same in elementary 32-bit torch operations where
it is false; ``exact`` is the definition in 64 bits, sequence by sequence.

A case's lengths follow from its own ``ragged`` number: ``batch`` sequences with ``new_low``..``new`` new
tokens behind ``past_low``..``past`` tokens that the cache holds already.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6
THETA = 1e6


def listed():
    model = {"heads": 32, "kv_heads": 8, "dim": 128, "type": "bf16"}  # the 8B backbone on one GPU
    shard = {"heads": 4, "kv_heads": 1, "dim": 128, "type": "bf16"}   # its shard at TP = 8
    return [
        # one decode step of a few requests: the smallest write, latency alone
        {"name": "write_step_b4", "op": "write", **model, "batch": 4, "new_low": 1, "new": 1, "past_low": 255,
         "past": 4095, "page": 64, "ragged": 1},
        # a batch of admitted prompts, 4 thousand rows of q|k|v
        {"name": "write_prompts_4k", "op": "write", **model, "batch": 9, "new_low": 130, "new": 770, "past_low": 0,
         "past": 0, "page": 64, "ragged": 2},
        # the batch-1 decode step at its usual context: few bytes, so the split and the join show
        {"name": "step_b1_2k", "op": "decode", **model, "batch": 1, "new_low": 1, "new": 1, "past_low": 2047,
         "past": 2047, "page": 64, "ragged": 3},
        # one long-form request
        {"name": "step_b1_32k", "op": "decode", **model, "batch": 1, "new_low": 1, "new": 1, "past_low": 32748,
         "past": 32748, "page": 128, "ragged": 4},
        # the ragged batched step of the decode sweep on one of eight GPUs, small pages
        {"name": "step_b64_shard", "op": "decode", **shard, "batch": 64, "new_low": 1, "new": 1, "past_low": 255,
         "past": 4095, "page": 16, "ragged": 5},
        # the largest step: 128 ragged requests on one GPU
        {"name": "step_b128", "op": "decode", **model, "batch": 128, "new_low": 1, "new": 1, "past_low": 255,
         "past": 4095, "page": 64, "ragged": 6},
        # one short sentence, latency alone
        {"name": "prompt_b1_33", "op": "packed", **model, "batch": 1, "new_low": 33, "new": 33, "past_low": 0,
         "past": 0, "causal": True, "ragged": 7},
        # sixteen prompts of 1 to 1024 tokens admitted together
        {"name": "prompts_b16", "op": "packed", **model, "batch": 16, "new_low": 1, "new": 1024, "past_low": 0,
         "past": 0, "causal": True, "ragged": 8},
        # bidirectional windows of an encoder: half precision, 64-wide heads, more keys than queries
        {"name": "windows_fp16_d64", "op": "packed", "heads": 16, "kv_heads": 16, "dim": 64, "type": "fp16",
         "batch": 12, "new_low": 100, "new": 750, "past_low": 0, "past": 501, "causal": False, "ragged": 9},
        # the largest prompt: long-form text with a reference voice
        {"name": "prompt_8k", "op": "packed", **model, "batch": 1, "new_low": 8191, "new": 8191, "past_low": 0,
         "past": 0, "causal": True, "ragged": 10},
        # chunks of prompts behind what the cache already holds of them
        {"name": "chunks_b4", "op": "prompt", **model, "batch": 4, "new_low": 190, "new": 700, "past_low": 500,
         "past": 4000, "page": 64, "causal": True, "ragged": 11},
        # a short continuation of one long request: few rows, a long axis
        {"name": "chunk_b1_16k", "op": "prompt", **model, "batch": 1, "new_low": 48, "new": 48, "past_low": 16001,
         "past": 16001, "page": 128, "causal": True, "ragged": 12},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    largest = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    while True:
        case = _drawn(rng)
        new, total = lengths(case)
        padded = case["batch"] * case["heads"] * max(new) * max(total)
        if all(work(case)[k] <= largest[k] for k in largest) and padded <= 2.2e9:
            return case


def _drawn(rng):
    op = rng.choice(["write", "decode", "decode", "packed", "packed", "prompt"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    case = {"op": op, "kv_heads": kv_heads, "heads": kv_heads * rng.choice([1, 2, 3, 4, 7, 8]),
            "dim": rng.choice([64, 128, 128]), "type": rng.choice(["bf16", "bf16", "fp16"]),
            "ragged": rng.randrange(1, 1 << 20)}
    if op != "packed":
        case["page"] = rng.choice([16, 32, 64, 128, 256])
    if op == "decode":
        case["batch"] = _log(rng, 1, 128)
        case["past"] = _log(rng, 1, min(40000, 500000 // case["batch"]))
        return case | {"new_low": 1, "new": 1, "past_low": rng.randrange(case["past"])}
    case["batch"] = _log(rng, 1, 40)
    case["new"] = _log(rng, 1, 8191)
    case["new_low"] = rng.randrange(1, case["new"] + 1)
    case["past"] = 0 if rng.random() < 0.4 else _log(rng, 1, 16000)
    case["past_low"] = rng.randrange(case["past"] + 1)
    if op != "write":
        case["causal"] = op == "prompt" or rng.random() < 0.7
    return case


def lengths(case):
    """(new tokens, all tokens) of each sequence."""
    r = random.Random(case["ragged"])
    new = [r.randint(case["new_low"], case["new"]) for _ in range(case["batch"])]
    return new, [n + r.randint(case["past_low"], case["past"]) for n in new]


def _rows(case):
    """Rows of the token buffers: the packed tokens, rounded up to a bucket of 16 as a server pads them."""
    new, _ = lengths(case)
    return sum(new) if case["op"] in ("decode",) or max(new) == 1 else -(-sum(new) // 16) * 16


def _starts(lens, dev):
    return torch.tensor([0] + lens, device=dev).cumsum(0).to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt, nq, nkv, d = TYPES[case["type"]], case["heads"], case["kv_heads"], case["dim"]
    new, total = lengths(case)
    t = _rows(case)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=dt)

    s = {"case": case, "max_new": max(new), "max_total": max(total), "cu": _starts(new, dev),
         "lens": torch.tensor(total, device=dev, dtype=torch.int32)}
    if case["op"] == "packed":
        # q, k and v as the q|k|v projection leaves them, where both have the same rows
        if new == total:
            qkv = normal(t, nq + 2 * nkv, d)
            s |= {"q": qkv[:, :nq], "k": qkv[:, nq:nq + nkv], "v": qkv[:, nq + nkv:], "cu_k": s["cu"]}
        else:
            s |= {"q": normal(t, nq, d), "k": normal(sum(total), nkv, d), "v": normal(sum(total), nkv, d),
                  "cu_k": _starts(total, dev)}
        s["out"] = torch.zeros(t, nq, d, device=dev, dtype=dt)
    else:
        # pages in the order in which requests came and went
        page = case["page"]
        need = [-(-n // page) for n in total]
        count = sum(need) + 3
        table = torch.zeros(case["batch"], max(need), dtype=torch.int32)
        order = torch.randperm(count, generator=g, device=dev).to(torch.int32).cpu()
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        s |= {"table": table.to(dev), "k": normal(count, nkv, page, d), "v": normal(count, nkv, page, d)}
        if case["op"] == "write":
            angle = (torch.arange(max(total), device=dev, dtype=torch.float64)[:, None]
                     * THETA ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)).repeat(1, 2)
            s |= {"qkv": normal(t, (nq + 2 * nkv) * d), "cos": angle.cos().to(dt), "sin": angle.sin().to(dt),
                  "q_weight": (1 + 0.02 * normal(d).float()).to(dt), "k_weight": (1 + 0.02 * normal(d).float()).to(dt),
                  "q": torch.zeros(t, nq, d, device=dev, dtype=dt)}
        else:
            s["q"] = normal(t, nq, d)
            s["out"] = torch.zeros(t, nq, d, device=dev, dtype=dt)
    return s


def run(state):
    return (_kernels if own else _plain)(state)


# ------------------------------------------------------------------ the framework's calls
def _kernels(s):
    k = _framework()
    op = s["case"]["op"]
    if op == "write":
        q = k.qk_rope_paged(s["qkv"], s["q_weight"], s["k_weight"], s["cos"], s["sin"], s["k"], s["v"], s["table"],
                            s["lens"], s["cu"], EPS, out=s["q"])
        return {"q": q, "k_pages": s["k"], "v_pages": s["v"]}
    if op == "decode":
        return k.paged_attention_decode(s["q"], s["k"], s["v"], s["table"], s["lens"], out=s["out"])
    if op == "prompt":
        return k.paged_attention_prompt(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu"], out=s["out"])
    return k.packed_attention(s["q"], s["k"], s["v"], s["cu"], s["cu_k"], causal=s["case"]["causal"], out=s["out"])


def _framework():
    root = str(Path(__file__).resolve().parent.parent / "moss-tts-optimized_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from moss_tts._runtime import kernels
    return kernels


# ------------------------------------------------------------------ the plain forms
def _plain(s):
    op, cu = s["case"]["op"], s["cu"]
    rows = torch.arange(s["q"].shape[0], device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), rows.to(cu.dtype), right=True)  # the sequence of each row
    live = seq < s["lens"].numel()
    seq = seq.clamp(max=s["lens"].numel() - 1)
    index = rows - cu[seq]  # its place among the new tokens
    if op == "write":
        return _plain_write(s, seq[live], index[live], rows[live])
    lens_q, lens_k = cu.diff(), s["lens"]
    padded = torch.arange(s["max_new"], device=cu.device)
    q = s["q"].float()[(cu[:-1, None] + padded).clamp(max=s["q"].shape[0] - 1)]
    keys = torch.arange(s["max_total"], device=cu.device)
    if op == "packed":
        at = (s["cu_k"][:-1, None] + keys).clamp(max=s["k"].shape[0] - 1)
        k, v = s["k"].float()[at], s["v"].float()[at]
    else:
        page = s["k"].shape[2]
        ids = s["table"][:, (keys // page)]
        k, v = s["k"].float()[ids, :, keys % page], s["v"].float()[ids, :, keys % page]
    o = _plain_attention(q, k, v, lens_q, lens_k, s["case"].get("causal", True))
    s["out"].copy_(torch.where(live[:, None, None], o[seq, index.clamp(min=0, max=s["max_new"] - 1)],
                               s["out"].float()))
    return s["out"]


def _plain_attention(q, k, v, lens_q, lens_k, causal):
    """softmax(q k^T / sqrt(d)) v of padded [B, rows, heads, d] in 32 bits; the last query sits at the last key."""
    b, lq, nq, d = q.shape
    lk, nkv = k.shape[1:3]
    q = q.view(b, lq, nkv, nq // nkv, d).permute(0, 2, 3, 1, 4).reshape(b, nkv, -1, d)
    score = (q @ k.permute(0, 2, 3, 1)).view(b, nkv, nq // nkv, lq, lk).mul_(d ** -0.5)
    key = torch.arange(lk, device=q.device)
    keep = key < lens_k[:, None, None]
    if causal:
        keep = keep & (key <= torch.arange(lq, device=q.device)[:, None] + (lens_k - lens_q)[:, None, None])
    score.masked_fill_(~keep[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(b, nkv, -1, lk) @ v.permute(0, 2, 1, 3)
    o = o.view(b, nkv, nq // nkv, lq, d) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(b, lq, nq, d)


def _plain_write(s, seq, index, rows):
    nq, nkv, page, d = s["q"].shape[1], *s["k"].shape[1:]
    position = (s["lens"] - s["cu"].diff())[seq] + index
    x = s["qkv"][rows].float().view(rows.numel(), nq + 2 * nkv, d)
    cos, sin = s["cos"][position].float()[:, None], s["sin"][position].float()[:, None]

    def rotated(x, weight):
        x = x * (x.square().mean(-1, keepdim=True) + EPS).rsqrt() * weight.float()
        return x * cos + torch.cat((-x[..., d // 2:], x[..., :d // 2]), -1) * sin

    ids, offset = s["table"][seq, position // page], position % page
    s["q"][rows] = rotated(x[:, :nq], s["q_weight"]).to(s["q"].dtype)
    s["k"][ids, :, offset] = rotated(x[:, nq:nq + nkv], s["k_weight"]).to(s["k"].dtype)
    s["v"][ids, :, offset] = x[:, nq + nkv:].to(s["v"].dtype)
    return {"q": s["q"], "k_pages": s["k"], "v_pages": s["v"]}


# ------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    new, total = lengths(case)
    if case["op"] == "write":
        return _exact_write(s, new, total)
    out = s["out"].double()
    first_q = first_k = 0
    for b, (n, m) in enumerate(zip(new, total)):
        if case["op"] == "packed":
            k, v = (s[x][first_k:first_k + m].double() for x in "kv")
        else:
            ids = s["table"][b, :-(-m // case["page"])].long()
            k, v = (s[x][ids].transpose(1, 2).reshape(-1, case["kv_heads"], case["dim"])[:m].double() for x in "kv")
        for h in range(case["heads"]):
            j = h // (case["heads"] // case["kv_heads"])
            score = s["q"][first_q:first_q + n, h].double() @ k[:, j].t() / math.sqrt(case["dim"])
            if case.get("causal", True):
                score += torch.full((n, m), -math.inf, device=score.device, dtype=score.dtype).triu(m - n + 1)
            out[first_q:first_q + n, h] = torch.softmax(score, -1) @ v[:, j]
        first_q, first_k = first_q + n, first_k + m
    return out


def _exact_write(s, new, total):
    case = s["case"]
    nq, nkv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    q, kp, vp = s["q"].double(), s["k"].double(), s["v"].double()
    half, first = d // 2, 0
    for b, (n, m) in enumerate(zip(new, total)):
        place = torch.arange(m - n, m, device=q.device)
        x = s["qkv"][first:first + n].double().view(n, -1, d)
        w = torch.cat((s["q_weight"].double().expand(nq, d), s["k_weight"].double().expand(nkv, d)))
        y = x[:, :nq + nkv] / torch.sqrt((x[:, :nq + nkv] ** 2).sum(-1, keepdim=True) / d + EPS) * w
        c, z = s["cos"][place].double().view(n, 1, d), s["sin"][place].double().view(n, 1, d)
        r = torch.empty_like(y)
        r[..., :half] = y[..., :half] * c[..., :half] - y[..., half:] * z[..., :half]
        r[..., half:] = y[..., half:] * c[..., half:] + y[..., :half] * z[..., half:]
        q[first:first + n] = r[:, :nq]
        ids = s["table"][b].long()[place // page]
        kp[ids, :, place % page] = r[:, nq:]
        vp[ids, :, place % page] = x[:, nq + nkv:]
        first += n
    return {"q": q, "k_pages": kp, "v_pages": vp}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    nq, nkv, d = case["heads"], case["kv_heads"], case["dim"]
    new, total = lengths(case)
    rows, cached = sum(new), sum(total)
    ints = 4 * (2 * case["batch"] + 1)
    if case["op"] != "packed":
        ints += 4 * sum(-(-n // case["page"]) for n in (new if case["op"] == "write" else total))
    if case["op"] == "write":  # q|k|v in, q, k and v out, a row of cos and of sin for each position
        places = len({p for n, m in zip(new, total) for p in range(m - n, m)})
        return {"bytes": 4 * rows * (nq + 2 * nkv) * d + 4 * places * d + 4 * d + ints,
                "flops": rows * (nq + nkv) * d * 7}
    pairs = sum(n * m - (n * (n - 1) // 2 if case.get("causal", True) else 0) for n, m in zip(new, total))
    return {"bytes": 4 * rows * nq * d + 4 * cached * nkv * d + ints, "flops": 4 * pairs * nq * d}
