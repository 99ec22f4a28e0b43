"""The serving-step operators and their measured cases: position rotation, append to a paged KV
cache with the rotation applied on the way, and attention of a batch over a shared prefix and the
sequences' own tails.

Each case is a dict of plain values; `prepare` makes a user's inputs on the GPU from a seed, `run`
is one pass (the plain torch form, or the framework's call where `own` is true), `exact` the
operator's definition in 64 bits, `work` the bytes and operations one pass cannot do without.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
# Container bytes over tight BF16 bytes of K and V with the distribution that prefix_kv() draws.
XKV_RATIO = 0.755


def _kvx():
    """The framework's Python binding."""
    path = os.path.join(ROOT, "compressed-kv-attention_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import kvexp_b200
    return kvexp_b200


# ---- cases -------------------------------------------------------------------------------------

def _attend(name, batch, hq, hkv, dim, prefix, tail, page, layout="nhd", kind="pages", dtype="bf16"):
    return {"name": name, "op": "attend", "batch": batch, "hq": hq, "hkv": hkv, "dim": dim, "prefix": prefix,
            "tail": tail, "page": page, "layout": layout, "kind": kind, "dtype": dtype}


def _append(name, tokens, seqs, hq, hkv, dim, rot, axes, interleaved, page, layout, dtype):
    return {"name": name, "op": "append", "tokens": tokens, "seqs": seqs, "hq": hq, "hkv": hkv, "dim": dim,
            "rot": rot, "axes": axes, "interleaved": interleaved, "page": page, "layout": layout, "dtype": dtype}


def _rotate(name, tokens, heads, dim, rot, axes, interleaved, inverse, dtype):
    return {"name": name, "op": "rotate", "tokens": tokens, "heads": heads, "dim": dim, "rot": rot, "axes": axes,
            "interleaved": interleaved, "inverse": inverse, "dtype": dtype}


def listed():
    return [
        # one generated token of one conversation goes into the cache: launch latency is all of it
        _append("append_token", 1, 1, 14, 2, 64, 64, 1, False, 16, "nhd", "bf16"),
        # the prompts of a batch, ragged, in one prefill call
        _append("append_prompts", 16384, 11, 32, 8, 128, 128, 1, False, 64, "hnd", "bf16"),
        # queries of video patches: positions in time, height and width
        _rotate("rotate_video", 5061, 14, 64, 64, 3, False, False, "bf16"),
        # the gradient of a partial rotation of adjacent pairs, a whole training batch
        _rotate("rotate_grad", 32768, 32, 128, 64, 1, True, True, "fp16"),
        # two requests behind a short system prompt: the smallest attention call
        _attend("attend_small", 2, 14, 2, 64, 1000, 64, 16),
        # a chat server's batch behind an 8K prompt
        _attend("attend_chat", 16, 14, 2, 64, 8192, 512, 16),
        # a large batch behind a 32K prefix, tails about as many bytes as the prefix
        _attend("attend_batch", 64, 32, 8, 128, 32768, 1024, 64),
        # a few agents behind one very long document; FP16, pages of an odd multiple, heads outermost
        _attend("attend_document", 7, 32, 8, 128, 131072, 777, 48, layout="hnd", dtype="fp16"),
        # the widest heads, a prefix that ends inside a page and a tile
        _attend("attend_wide", 5, 32, 8, 256, 20001, 300, 128),
        # no grouped heads, narrow; most of the work is in the tails
        _attend("attend_tails", 33, 16, 16, 32, 4097, 2049, 32),
        # the chat batch behind a long prompt that is kept compressed
        _attend("attend_xkv_chat", 16, 14, 2, 64, 32768, 256, 16, kind="xkv"),
        # the larger model's batch behind a compressed prefix, odd length
        _attend("attend_xkv_batch", 32, 32, 8, 128, 32731, 512, 64, kind="xkv"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {"bytes": max(work(c)["bytes"] for c in listed()), "flops": max(work(c)["flops"] for c in listed())}
    while True:
        c = _draw_one(rng)
        w = work(c)
        # the plain form gathers every tail at the longest one's length
        padded = 0 if c["op"] != "attend" else 4 * c["batch"] * c["tail"] * c["hkv"] * c["dim"]
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and padded <= most["bytes"]:
            return c


def _draw_one(rng):
    hq, hkv, dim = rng.choice([(14, 2, 64), (32, 8, 128), (32, 8, 256), (16, 16, 32), (8, 1, 128), (12, 4, 64),
                               (20, 2, 128), (6, 6, 64), (9, 3, 32)])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    page = rng.choice([1, 16, 16, 32, 48, 64, 128])
    layout = rng.choice(["nhd", "hnd"])
    kind = rng.random()
    if kind < 0.6:
        prefix = 0 if rng.random() < 0.08 else _log_int(rng, 1, 131072)
        tail = 0 if rng.random() < 0.08 else _log_int(rng, 1, 4096)
        xkv = prefix > 0 and rng.random() < 0.35
        c = _attend("", _log_int(rng, 1, 96), hq, hkv, dim, prefix, tail, page, layout,
                    "xkv" if xkv else "pages", "bf16" if xkv else dtype)
    else:
        axes = rng.choice([1, 1, 3, 2])
        rot = rng.choice([dim, dim, dim // 2, dim // 4 * 3])
        tokens = _log_int(rng, 1, 20000)
        if kind < 0.85:
            c = _append("", tokens, max(1, min(tokens, _log_int(rng, 1, 200))), hq, hkv, dim, rot, axes,
                        rng.random() < 0.4, page, layout, dtype)
        else:
            c = _rotate("", tokens, rng.choice([hq, hkv]), dim, rot, axes, rng.random() < 0.4, rng.random() < 0.5, dtype)
    del c["name"]
    return c


def tail_lens(case):
    """Tokens in each sequence's own pages: ragged, the first the longest, the last of three or more empty."""
    n, t = case["batch"], case["tail"]
    lens = [max(0, t - int(t * ((i * 0.6180339887) % 1.0))) for i in range(n)]
    if n >= 3:
        lens[-1] = 0
    return lens


def work(case):
    d = case["dim"]
    if case["op"] == "rotate":
        n = case["tokens"] * case["heads"]
        return {"bytes": 4 * n * d, "flops": 3 * n * case["rot"]}
    if case["op"] == "append":
        t = case["tokens"]
        return {"bytes": 4 * t * (case["hq"] + 2 * case["hkv"]) * d, "flops": 3 * t * (case["hq"] + case["hkv"]) * case["rot"]}
    b, tails = case["batch"], sum(tail_lens(case))
    prefix = 4 * case["prefix"] * case["hkv"] * d * (XKV_RATIO if case["kind"] == "xkv" else 1.0)
    rows = 4 * b * case["hq"] * d + 4 * b * case["hq"]
    return {"bytes": prefix + 4 * tails * case["hkv"] * d + rows, "flops": 4 * case["hq"] * d * (b * case["prefix"] + tails)}


# ---- inputs ------------------------------------------------------------------------------------

def _tables(case, dev):
    """cos and sin of every position up to 32768, as a model keeps them."""
    half = case["rot"] // 2
    inv = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
    a = torch.arange(32768, device=dev, dtype=torch.float64)[:, None] * inv[None, :]
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def _axes(case, dev):
    """The axis of each pair: runs of pairs, the first shorter, as multimodal models divide them."""
    half, n = case["rot"] // 2, case["axes"]
    if n == 1:
        return torch.zeros(half, dtype=torch.uint8, device=dev)
    cut = [half // 4 + (half - half // 4) * i // (n - 1) for i in range(n)]
    at = torch.arange(half, device=dev)
    return sum((at >= c).to(torch.uint8) for c in cut[:-1])


def _positions(case, n, gen, dev):
    """[axes, n] positions: running along a text from some start, or the places of a grid of patches."""
    start = int(torch.randint(0, 4000, (1,), generator=gen, device=dev))
    t = torch.arange(n, device=dev)
    if case["axes"] == 1:
        p = (start + t)[None] % 32768
    else:
        w = 23
        p = torch.stack([start + t // (w * w), start + (t // w) % w, start + t % w])[-case["axes"]:] % 32768
    return p.to(torch.int32).contiguous()


def _pool(case, n_pages, gen, dev, dtype):
    """K and V pools [pages, tokens, heads, dim] (heads outside tokens in memory for "hnd") with old contents."""
    h, d, pg = case["hkv"], case["dim"], case["page"]
    scale = torch.exp2(torch.randint(-2, 3, (h, 1, d), generator=gen, device=dev).float() / 2)
    out = []
    for i in range(2):
        x = torch.randn((n_pages, h, pg, d), generator=gen, device=dev, dtype=torch.float32)
        x = (x * scale if i == 0 else x * 0.5).to(dtype)
        out.append(x.transpose(1, 2) if case["layout"] == "hnd" else x.transpose(1, 2).contiguous())
    return out


def _prefix_kv(case, gen, dev):
    """K and V [heads, tokens, dim] BF16 of a prefix: per-channel scales as keys have them, 0.3 % of outliers."""
    shape = (case["hkv"], case["prefix"], case["dim"])
    scale = torch.exp2(torch.randint(-2, 3, (case["hkv"], 1, case["dim"]), generator=gen, device=dev).float() / 2)
    out = []
    for i in range(2):
        x = torch.randn(shape, generator=gen, device=dev)
        x *= scale if i == 0 else 0.5
        far = torch.rand(shape, generator=gen, device=dev) < 0.003
        out.append(torch.where(far, x / 512, x).to(torch.bfloat16).contiguous())
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dtype = TYPES[case["dtype"]]
    s = {"case": case, "dtype": dtype}
    if case["op"] == "attend":
        _prepare_attend(case, s, gen, dev, dtype)
        return s
    s["cos"], s["sin"] = _tables(case, dev)
    s["axis"] = _axes(case, dev)
    n, d = case["tokens"], case["dim"]
    s["pos"] = _positions(case, n, gen, dev)
    if case["op"] == "rotate":
        s["x"] = torch.randn((n, case["heads"], d), generator=gen, device=dev).to(dtype)
        s["out"] = torch.empty_like(s["x"])
    else:
        # q, k and v are views of the projection's one output
        hq, hkv, page = case["hq"], case["hkv"], case["page"]
        qkv = torch.randn((n, hq + 2 * hkv, d), generator=gen, device=dev).to(dtype)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["q_out"] = torch.empty((n, hq, d), device=dev, dtype=dtype)
        # sequence i holds the i-th run of tokens, beginning inside its first page; every 61st of many is padding
        per = -(-n // case["seqs"])
        seq, at = torch.arange(n, device=dev) // per, torch.arange(n, device=dev) % per
        first = torch.randint(0, page, (case["seqs"],), generator=gen, device=dev)
        need = -(-(per + page) // page)
        n_pages = case["seqs"] * need + 3
        perm = torch.randperm(n_pages, generator=gen, device=dev)
        where = first[seq] + at
        slots = perm[seq * need + where // page] * page + where % page
        s["slots"] = torch.where(torch.arange(n, device=dev) % 61 == 60, torch.full_like(slots, -1), slots).to(torch.int64)
        s["k_pool"], s["v_pool"] = _pool(case, n_pages, gen, dev, dtype)
    if own:
        kvx = _kvx()
        heads = (case["hq"], case["hkv"]) if case["op"] == "append" else (case["heads"], case["heads"])
        s["batch"] = kvx.Batch(1, heads[0], heads[1], d, dtype=case["dtype"])
        s["rope"] = kvx.Rope(s["cos"], s["sin"], axis=s["axis"] if case["axes"] > 1 else None, n_axes=case["axes"],
                             interleaved=case["interleaved"])
        if case["op"] == "append":
            s["pages"] = kvx.Pages(s["k_pool"], s["v_pool"])
    return s


def _prepare_attend(case, s, gen, dev, dtype):
    b, d, page, hkv = case["batch"], case["dim"], case["page"], case["hkv"]
    lens = tail_lens(case)
    n_table = max(1, -(-case["tail"] // page))
    xkv = case["kind"] == "xkv"
    n_prefix = 0 if xkv else -(-case["prefix"] // page)
    n_pages = n_prefix + b * n_table + 2
    s["k_pool"], s["v_pool"] = _pool(case, n_pages, gen, dev, dtype)
    perm = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
    s["prefix_table"] = perm[:n_prefix].contiguous()
    s["table"] = perm[n_prefix:n_prefix + b * n_table].reshape(b, n_table).contiguous()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    # queries whose scores spread over a few units, as after training
    s["q"] = (torch.randn((b, case["hq"], d), generator=gen, device=dev) * 1.2).to(dtype)
    s["scale"] = d ** -0.5
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty((b, case["hq"]), device=dev, dtype=torch.float32)
    if xkv:
        s["k_prefix"], s["v_prefix"] = _prefix_kv(case, gen, dev)
    if own:
        kvx = _kvx()
        s["batch"] = kvx.Batch(b, case["hq"], hkv, d, dtype=case["dtype"])
        s["pages"] = kvx.Pages(s["k_pool"], s["v_pool"])
        if xkv:
            s["prefix"] = kvx.Prefix.encode(s["k_prefix"], s["v_prefix"])


# ---- one pass ----------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        stream = torch.cuda.current_stream().cuda_stream
        if case["op"] == "rotate":
            s["batch"].rotate(s["x"], s["pos"], s["rope"], s["out"], inverse=case["inverse"], stream=stream)
            return s["out"]
        if case["op"] == "append":
            s["batch"].append(s["q"], s["k"], s["v"], s["pos"], s["rope"], s["slots"], s["pages"], s["q_out"], stream=stream)
            return {"q": s["q_out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
        shared = {"prefix": s["prefix"]} if case["kind"] == "xkv" else {
            "prefix_table": s["prefix_table"], "prefix_len": case["prefix"]}
        s["batch"].attend(s["q"], s["out"], s["pages"], s["table"], s["lens"], case["tail"], scale=s["scale"],
                          lse=s["lse"], stream=stream, **shared)
        return {"out": s["out"], "lse": s["lse"]}
    if case["op"] == "rotate":
        return _plain_rotate(s["x"], s, case["inverse"])
    if case["op"] == "append":
        return _plain_append(s)
    return _plain_attend(s)


def _plain_rotate(x, s, inverse=False):
    case = s["case"]
    half = case["rot"] // 2
    pos = s["pos"].long()[s["axis"].long()].T                    # [tokens, half]
    at = torch.arange(half, device=x.device)
    c, w = s["cos"][pos, at][:, None], s["sin"][pos, at][:, None]
    if inverse:
        w = -w
    y = x.float()
    r, rest = y[..., :case["rot"]], y[..., case["rot"]:]
    if case["interleaved"]:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * c - b * w, b * c + a * w], dim=-1).flatten(-2)
    else:
        a, b = r[..., :half], r[..., half:]
        r = torch.cat([a * c - b * w, b * c + a * w], dim=-1)
    return torch.cat([r, rest], dim=-1).to(x.dtype)


def _plain_append(s):
    kept = s["slots"] >= 0
    slot = s["slots"][kept]
    page = s["case"]["page"]
    s["k_pool"][slot // page, slot % page] = _plain_rotate(s["k"], s)[kept]
    s["v_pool"][slot // page, slot % page] = s["v"][kept]
    return {"q": _plain_rotate(s["q"], s), "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_attend(s):
    case = s["case"]
    b, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["dim"]
    q = s["q"].float().view(b, hkv, hq // hkv, d) * s["scale"]
    if case["kind"] == "xkv":
        kp, vp = s["k_prefix"].float(), s["v_prefix"].float()
    else:
        kp, vp = (p[s["prefix_table"].long()].flatten(0, 1)[:case["prefix"]].transpose(0, 1).float() for p in (s["k_pool"], s["v_pool"]))
    kt, vt = (p[s["table"].long()].flatten(1, 2)[:, :case["tail"]].permute(0, 2, 1, 3).float() for p in (s["k_pool"], s["v_pool"]))
    rows = q.permute(1, 0, 2, 3).reshape(hkv, -1, d)              # [hkv, batch * group, d]
    sp = (rows @ kp.transpose(1, 2)).view(hkv, b, hq // hkv, -1).transpose(0, 1)
    st = q @ kt.transpose(2, 3)                                   # [batch, hkv, group, tail]
    past = torch.arange(case["tail"], device=q.device)[None] >= s["lens"][:, None]
    st = st.masked_fill(past[:, None, None], -math.inf)
    sc = torch.cat([sp, st], dim=-1)
    none = torch.full(sc.shape[:-1] + (1,), -math.inf, device=q.device)
    m = torch.cat([sc, none], dim=-1).amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -math.inf, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    n = sp.shape[-1]
    o = (p[..., :n].transpose(0, 1).reshape(hkv, -1, n) @ vp).view(hkv, b, hq // hkv, d).transpose(0, 1) + p[..., n:] @ vt
    o = torch.where(l > 0, o / l, torch.zeros_like(o))
    return {"out": o.reshape(b, hq, d).to(s["dtype"]), "lse": (m + torch.log(l)).reshape(b, hq)}


# ---- 64 bits -----------------------------------------------------------------------------------

def _exact_rotate(x, s, sign):
    case = s["case"]
    x = x.double().clone()
    half, rot = case["rot"] // 2, case["rot"]
    for i in range(half):
        p = s["pos"][int(s["axis"][i])].long()
        c, w = s["cos"][p, i].double()[:, None], sign * s["sin"][p, i].double()[:, None]
        u, v = (2 * i, 2 * i + 1) if case["interleaved"] else (i, rot - half + i)
        a, b = x[..., u].clone(), x[..., v].clone()
        x[..., u] = a * c - b * w
        x[..., v] = a * w + b * c
    return x


def exact(case, seed):
    """The operators' definitions in 64 bits, one sequence and head at a time."""
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(s["x"], s, -1.0 if case["inverse"] else 1.0)
    if case["op"] == "append":
        page, k = case["page"], _exact_rotate(s["k"], s, 1.0)
        kp, vp = s["k_pool"].double(), s["v_pool"].double()
        keep = torch.nonzero(s["slots"] >= 0).flatten()
        slot = s["slots"][keep]
        kp.index_put_((slot // page, slot % page), k[keep])
        vp.index_put_((slot // page, slot % page), s["v"][keep].double())
        return {"q": _exact_rotate(s["q"], s, 1.0), "k_pool": kp, "v_pool": vp}
    b, hq, hkv, d, page = case["batch"], case["hq"], case["hkv"], case["dim"], case["page"]
    out = torch.zeros((b, hq, d), dtype=torch.float64, device=s["q"].device)
    lse = torch.full((b, hq), -math.inf, dtype=torch.float64, device=s["q"].device)
    lens = tail_lens(case)
    for h in range(hkv):
        heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
        if case["kind"] == "xkv":
            kp, vp = s["k_prefix"][h].double(), s["v_prefix"][h].double()
        else:
            t = s["prefix_table"].long()
            kp, vp = (x[t, :, h].reshape(-1, d)[:case["prefix"]].double() for x in (s["k_pool"], s["v_pool"]))
        for i in range(b):
            t = s["table"][i, :-(-lens[i] // page)].long()
            kt, vt = (x[t, :, h].reshape(-1, d)[:lens[i]].double() for x in (s["k_pool"], s["v_pool"]))
            if case["prefix"] + lens[i] == 0:
                continue
            q = s["q"][i, heads].double() * s["scale"]
            sc = torch.cat([q @ kp.T, q @ kt.T], dim=1)
            lse[i, heads] = torch.logsumexp(sc, 1)
            w = torch.softmax(sc, 1)
            out[i, heads] = w[:, :case["prefix"]] @ vp + w[:, case["prefix"]:] @ vt
    return {"out": out, "lse": lse}
