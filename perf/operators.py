"""Attention over a paged key-value cache, and the two operators that a program needs around it, as timed cases.

  append  the new tokens' keys, rotated by their positions, and values go into the pages of their sequences; the queries are
          rotated on the way (`ops.paged_append`). One token a sequence while decoding, whole prompts before that.
  decode  one new token a sequence attends to its sequence's pages (`ops.paged_attn_decode`).
  prompt  causal attention inside packed prompts of different lengths (`ops.prompt_attn`).

q, k and v are column ranges of one matrix, as a stacked projection leaves them. Pages lie in the cache in no order, and a row of
the page table is filled with -1 behind the sequence's last page.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_L2_BYTES = 126 << 20


def listed():
    return [
        # one token of a 7B-class model into a 32-bit cache: the smallest call, all latency
        dict(name="append_f32_step1", op="append", seqs=1, longest=512, ragged=False, step=True, heads=32, kv_heads=32,
             head_dim=128, page=16, act="f32", cache="f32"),
        # a serving batch decodes: one token for each of 48 sequences, grouped heads, 16-bit cache under 32-bit activations
        dict(name="append_f16_step48", op="append", seqs=48, longest=300, ragged=True, step=True, heads=32, kv_heads=8,
             head_dim=128, page=16, act="f32", cache="f16"),
        # a prompt of odd length on a small model with narrow heads
        dict(name="append_f16_prompt1", op="append", seqs=1, longest=1023, ragged=False, step=False, heads=16, kv_heads=16,
             head_dim=64, page=32, act="f32", cache="f16"),
        # several prompts admitted at once, 16-bit throughout
        dict(name="append_bf16_prompts", op="append", seqs=5, longest=6000, ragged=True, step=False, heads=32, kv_heads=8,
             head_dim=128, page=64, act="bf16", cache="bf16"),
        # one sequence just after a 512-token prompt, every head its own keys, 32-bit cache
        dict(name="decode_f32_one", op="decode", seqs=1, longest=513, ragged=False, heads=32, kv_heads=32, head_dim=128, page=16,
             act="f32", cache="f32"),
        # one sequence over a very long document: few rows, the work is along the length
        dict(name="decode_f16_long", op="decode", seqs=1, longest=100003, ragged=False, heads=32, kv_heads=8, head_dim=128,
             page=64, act="f32", cache="f16"),
        # a serving batch of very different lengths, a free slot among them
        dict(name="decode_bf16_batch64", op="decode", seqs=64, longest=8192, ragged=True, heads=32, kv_heads=8, head_dim=128,
             page=16, act="bf16", cache="bf16"),
        # many short conversations on a model with narrow heads
        dict(name="decode_f16_batch256", op="decode", seqs=256, longest=2047, ragged=True, heads=32, kv_heads=4, head_dim=64,
             page=32, act="f16", cache="f16"),
        # a question of a few words: latency
        dict(name="prompt_f16_short", op="prompt", seqs=1, longest=37, ragged=False, heads=32, kv_heads=8, head_dim=128,
             act="f16"),
        # a 512-token prompt of the 7B-class model with 32-bit activations
        dict(name="prompt_f32_512", op="prompt", seqs=1, longest=512, ragged=False, heads=32, kv_heads=32, head_dim=128,
             act="f32"),
        # a batch of prompts packed one behind the other
        dict(name="prompt_bf16_packed", op="prompt", seqs=24, longest=2048, ragged=True, heads=32, kv_heads=8, head_dim=128,
             act="bf16"),
        # one long document: the dense contraction
        dict(name="prompt_f16_16k", op="prompt", seqs=1, longest=16384, ragged=False, heads=32, kv_heads=8, head_dim=128,
             act="f16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "decode", "decode", "prompt", "prompt"))
    kv_heads = rng.choice((1, 2, 4, 5, 8, 16, 32))
    group = rng.choice([g for g in (1, 2, 3, 4, 7, 8, 16) if g * kv_heads <= 32])
    head_dim = 128 if rng.random() < 0.7 else 64
    act = rng.choice(sorted(_TYPES))
    cache = rng.choice(sorted(_TYPES)) if act == "f32" else act
    case = dict(op=op, heads=group * kv_heads, kv_heads=kv_heads, head_dim=head_dim, act=act)
    if op == "append":
        step = rng.random() < 0.5
        seqs = _log_int(rng, 1, 256) if step else _log_int(rng, 1, 12)
        row = head_dim * 2 * kv_heads * _BYTES[cache]
        if not step:
            row += head_dim * _BYTES[act] * (2 * group + 3) * kv_heads
        longest = _log_int(rng, 1, max(2, min(400 if step else 6000, 300000000 // row // seqs)))
        return dict(case, seqs=seqs, longest=longest, ragged=seqs > 1, step=step, page=rng.choice((1, 8, 16, 32, 64, 128)), cache=cache)
    if op == "decode":
        seqs = _log_int(rng, 1, 256)
        rows = min(120000, 500000000 // (2 * kv_heads * head_dim * _BYTES[cache]))   # keys of all sequences together
        return dict(case, seqs=seqs, longest=_log_int(rng, 1, max(2, rows // seqs)), ragged=seqs > 1 and rng.random() < 0.8,
                    page=rng.choice((1, 8, 16, 32, 64, 128)), cache=cache)
    seqs = _log_int(rng, 1, 32)
    return dict(case, seqs=seqs, longest=_log_int(rng, 1, min(8192, 24000 // seqs)), ragged=seqs > 1)


def _lengths(case):
    """Tokens of each sequence: spread over the logarithm, the longest one in the middle; in larger decode batches one slot is free."""
    n, longest = case["seqs"], case["longest"]
    if not case["ragged"]:
        return [longest] * n
    rng = random.Random(1000003 * n + longest)
    lens = [_log_int(rng, max(1, longest // 50), longest) for _ in range(n)]
    lens[n // 2] = longest
    if case["op"] == "decode" and n >= 8:
        lens[n // 3] = 0
    return lens


def _normal(shape, seed, dtype, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _tables(positions, head_dim):
    """cos and sin of every position's angles, [position][head_dim], both halves alike."""
    inv = 10000.0 ** (-torch.arange(0, head_dim, 2, dtype=torch.float64, device="cuda") / head_dim)
    ang = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv[None, :]
    ang = torch.cat((ang, ang), dim=1)
    return ang.cos().float(), ang.sin().float()


def _pages(case, lens, seed):
    """Page table of the sequences: their pages in no order, -1 behind the last one; and how many pages the cache has."""
    page = case["page"]
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3                                     # a few that nobody holds
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(1, max(need))
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return _ints(table), total


def _inputs(case, seed):
    lens = _lengths(case)
    h, kv, d, act = case["heads"], case["kv_heads"], case["head_dim"], _TYPES[case["act"]]
    x = dict(case=case, lens=lens, scale=1.0 / math.sqrt(d))
    if case["op"] == "decode":
        rows = case["seqs"]
    elif case["op"] == "append" and case["step"]:
        rows = case["seqs"]
    else:
        rows = sum(lens)
    qkv = _normal((rows, (h + 2 * kv) * d), seed, act, 1.25)
    x["q"] = qkv[:, :h * d].view(rows, h, d)
    x["k"] = qkv[:, h * d:(h + kv) * d].view(rows, kv, d)
    x["v"] = qkv[:, (h + kv) * d:].view(rows, kv, d)
    if case["op"] == "prompt":
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        x["starts"] = _ints(starts)
        return x
    x["table"], n_pages = _pages(case, lens, seed)
    shape = (n_pages, kv, case["page"], d)
    x["kc"] = _normal(shape, seed + 1_000_003, _TYPES[case["cache"]], 1.25)
    x["vc"] = _normal(shape, seed + 2_000_003, _TYPES[case["cache"]])
    if case["op"] == "decode":
        x["lens_d"] = _ints(lens)
        return x
    x["cos"], x["sin"] = _tables(max(max(lens), 1), d)
    if case["step"]:                                          # the newest position of each sequence
        x["seq_ids"], x["positions"] = _ints(list(range(rows))), _ints([n - 1 for n in lens])
    else:
        x["seq_ids"] = _ints([s for s, n in enumerate(lens) for _ in range(n)])
        x["positions"] = _ints([p for n in lens for p in range(n)])
    return x


def prepare(case, seed):
    """A model has a cache a layer: small caches come in several copies, and a pass takes the next one, so that what it reads
    is not in the L2 cache from the pass before."""
    x = _inputs(case, seed)
    if "kc" in x:
        nbytes = x["kc"].numel() * x["kc"].element_size() * 2
        copies = max(1, min(32, math.ceil(2 * _L2_BYTES / nbytes))) if case["op"] == "decode" else 1
        x["caches"] = [(x["kc"], x["vc"])] + [(x["kc"].clone(), x["vc"].clone()) for _ in range(copies - 1)]
        x["next"] = 0
    x["out"] = torch.empty(x["q"].shape, dtype=x["q"].dtype, device="cuda")
    if case["op"] == "append" and not case["step"]:           # a prompt's attention reads the rotated keys too
        x["k_out"] = torch.empty(x["k"].shape, dtype=x["k"].dtype, device="cuda")
    if own:
        from fuel_b200 import ops
        if case["op"] == "decode":
            x["workspace"] = ops.paged_attn_workspace(case["seqs"], case["heads"], case["kv_heads"], case["head_dim"], x["q"].device)
        elif case["op"] == "prompt":
            x["workspace"] = ops.prompt_attn_workspace(x["q"], x["k"])
    return x


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    x = x.float()
    lo, hi = x[..., :half], x[..., half:]
    return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), dim=-1)


def _append_plain(x):
    kc, vc = x["caches"][0]
    half = x["case"]["head_dim"] // 2
    pos, page = x["positions"].long(), x["case"]["page"]
    cos, sin = x["cos"][pos][:, None, :half], x["sin"][pos][:, None, :half]
    ids = x["table"][x["seq_ids"].long(), pos // page].long()
    q, k = _rotate(x["q"], cos, sin), _rotate(x["k"], cos, sin)
    x["out"].copy_(q)
    kc[ids, :, pos % page] = k.to(kc.dtype)
    vc[ids, :, pos % page] = x["v"].to(vc.dtype)
    if "k_out" not in x:
        return x["out"], kc, vc
    x["k_out"].copy_(k)
    return x["out"], x["k_out"], kc, vc


def _decode_plain(x):
    case, (kc, vc) = x["case"], x["caches"][x["next"]]
    x["next"] = (x["next"] + 1) % len(x["caches"])
    kv, d, group = case["kv_heads"], case["head_dim"], case["heads"] // case["kv_heads"]
    per = max(1, 300_000_000 // max(1, x["table"].shape[1] * case["page"] * kv * d))     # sequences at a time
    for a in range(0, case["seqs"], per):
        table, lens = x["table"][a:a + per], x["lens_d"][a:a + per]
        n = table.shape[0]
        ids = table.clamp(min=0).long()
        k = kc[ids].float().transpose(1, 2).reshape(n, kv, -1, d)
        v = vc[ids].float().transpose(1, 2).reshape(n, kv, -1, d)
        q = x["q"][a:a + per].float().view(n, kv, group, d)
        s = (q @ k.transpose(2, 3)) * x["scale"]
        seen = torch.arange(k.shape[2], device="cuda") < lens[:, None]
        s = torch.where(seen[:, None, None, :], s, float("-inf"))
        top = s.amax(dim=-1, keepdim=True)
        p = torch.exp(s - torch.where(top.isinf(), 0.0, top))
        total = p.sum(dim=-1, keepdim=True)
        x["out"][a:a + per] = ((p @ v) / torch.where(total == 0, 1.0, total)).view(n, case["heads"], d)
    return x["out"]


def _prompt_plain(x):
    case = x["case"]
    h, kv, d = case["heads"], case["kv_heads"], case["head_dim"]
    at = 0
    for n in x["lens"]:
        q = x["q"][at:at + n].float().view(n, kv, h // kv, d).permute(1, 2, 0, 3)
        k = x["k"][at:at + n].float().transpose(0, 1)[:, None]
        v = x["v"][at:at + n].float().transpose(0, 1)[:, None]
        for a in range(0, n, 1024):
            b = min(n, a + 1024)
            s = (q[:, :, a:b] @ k[:, :, :b].transpose(2, 3)) * x["scale"]
            future = torch.arange(b, device="cuda")[None, :] > torch.arange(a, b, device="cuda")[:, None]
            s = s.masked_fill(future, float("-inf"))
            p = torch.exp(s - s.amax(dim=-1, keepdim=True))
            o = (p @ v[:, :, :b]) / p.sum(dim=-1, keepdim=True)
            x["out"][at + a:at + b] = o.permute(2, 0, 1, 3).reshape(b - a, h, d)
        at += n
    return x["out"]


def run(state):
    x, op = state, state["case"]["op"]
    if not own:
        return {"append": _append_plain, "decode": _decode_plain, "prompt": _prompt_plain}[op](x)
    from fuel_b200 import ops
    if op == "append":
        kc, vc = x["caches"][0]
        ops.paged_append(x["k"], x["v"], kc, vc, x["table"], x["positions"], x["cos"], x["sin"], seq_ids=x["seq_ids"], q=x["q"],
                         q_out=x["out"], k_out=x.get("k_out"))
        return (x["out"], x["k_out"], kc, vc) if "k_out" in x else (x["out"], kc, vc)
    if op == "decode":
        kc, vc = x["caches"][x["next"]]
        x["next"] = (x["next"] + 1) % len(x["caches"])
        return ops.paged_attn_decode(x["q"], kc, vc, x["table"], x["lens_d"], x["scale"], out=x["out"], workspace=x["workspace"])
    return ops.prompt_attn(x["q"], x["k"], x["v"], x["starts"], x["scale"], out=x["out"], workspace=x["workspace"])


def work(case):
    lens, d, h, kv = _lengths(case), case["head_dim"], case["heads"], case["kv_heads"]
    act = _BYTES[case["act"]]
    if case["op"] == "append":
        rows = len(lens) if case["step"] else sum(lens)
        distinct = len(set(lens)) if case["step"] else max(lens)          # rows of the two tables, of which a half is enough
        nbytes = rows * d * (act * (2 * h + 2 * kv + (0 if case["step"] else kv)) + 2 * kv * _BYTES[case["cache"]])
        return {"bytes": nbytes + rows * 12 + distinct * 2 * 4 * (d // 2), "flops": 3 * rows * d * (h + kv)}
    if case["op"] == "decode":
        keys = sum(lens)
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2 * keys * kv * d * _BYTES[case["cache"]] + 2 * len(lens) * h * d * act + 4 * (pages + len(lens)),
                "flops": 4 * keys * h * d}
    pairs = sum(n * (n + 1) // 2 for n in lens)
    return {"bytes": sum(lens) * d * act * (2 * h + 2 * kv), "flops": 4 * pairs * h * d}


def exact(case, seed):
    """The definitions in 64 bits: each head of each sequence by itself, its keys in order."""
    x = _inputs(case, seed)
    h, kv, d, page = case["heads"], case["kv_heads"], case["head_dim"], case.get("page")
    dev = x["q"].device
    if case["op"] == "append":
        half = d // 2

        def turned(t):
            c = x["cos"].double()[x["positions"].long()][:, :half].unsqueeze(1)
            s = x["sin"].double()[x["positions"].long()][:, :half].unsqueeze(1)
            out = torch.empty(t.shape, dtype=torch.float64, device=dev)
            out[..., :half] = t[..., :half].double() * c - t[..., half:].double() * s
            out[..., half:] = t[..., half:].double() * c + t[..., :half].double() * s
            return out

        kc, vc, k = x["kc"].double(), x["vc"].double(), turned(x["k"])
        slot = x["table"].long()[x["seq_ids"].long(), torch.div(x["positions"].long(), page, rounding_mode="floor")] * page
        slot = slot + x["positions"].long() % page
        for cache, new in ((kc, k), (vc, x["v"].double())):
            flat = cache.permute(0, 2, 1, 3).reshape(-1, kv, d).clone()
            flat[slot] = new
            cache.copy_(flat.view(-1, page, kv, d).permute(0, 2, 1, 3))
        return (turned(x["q"]), kc, vc) if case["step"] else (turned(x["q"]), k, kc, vc)
    out = torch.zeros(x["q"].shape, dtype=torch.float64, device=dev)
    at = 0
    for i, n in enumerate(x["lens"]):
        if n == 0:
            continue
        if case["op"] == "decode":
            ids = x["table"][i, :-(-n // page)].long()
            k = x["kc"][ids].permute(0, 2, 1, 3).reshape(-1, kv, d)[:n].double()
            v = x["vc"][ids].permute(0, 2, 1, 3).reshape(-1, kv, d)[:n].double()
            for j in range(kv):
                heads = slice(j * (h // kv), (j + 1) * (h // kv))
                w = torch.softmax(x["q"][i, heads].double() @ k[:, j].T * x["scale"], dim=-1)
                out[i, heads] = w @ v[:, j]
            continue
        rows = torch.arange(n, device=dev)
        for j in range(h):
            k, v = x["k"][at:at + n, j // (h // kv)].double(), x["v"][at:at + n, j // (h // kv)].double()
            for a in range(0, n, 4096):
                b = min(n, a + 4096)
                s = x["q"][at + a:at + b, j].double() @ k[:b].T * x["scale"]
                s[rows[None, :b] > rows[a:b, None]] = float("-inf")
                out[at + a:at + b, j] = torch.softmax(s, dim=-1) @ v[:b]
        at += n
    return out
