"""What the operators of a sampled decode step over an 8-bit KV cache cost.

Four operators, next to the fp16 paths of this package (same page layout, same
block tables, Qwen2.5-0.5B head shapes unless a case says otherwise):

* ``write``: the K and V rows of a decode or mixed pass, quantised into their
  pages with one scale per (page, K or V, kv head), and the pages that the pass
  touched read back (with the rotary embedding of q and k, or without);
* ``read``: positions [starts, lens) of sequences dequantised into a fp16 pool;
* ``attend``: decode attention over the 8-bit pages;
* ``sample``: a token per row of logits with temperature, top-k, top-p, min-p.

A page is 16 tokens. Its scale is the smallest power of two 2^e, -24 <= e <= 9,
with max |x| <= 127 * 2^e over the rows written so far (and never less than the
scale under which the page's older rows were stored); a code is x / scale
rounded to nearest even and clamped to +-127.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
D = 64


# ---- cases ---------------------------------------------------------------------


def listed():
    return [
        # one decode step of a small batch: eight rows, each into its own page
        {"name": "write decode 8", "op": "write", "mode": "decode", "batch": 8, "hkv": 2,
         "lo": 5, "hi": 2000, "tokens": 8, "rope": True, "wide": True},
        # a full mixed pass of the token budget: 32 ragged chunks behind ragged histories
        {"name": "write mixed 2048", "op": "write", "mode": "mixed", "batch": 32, "hkv": 2,
         "lo": 0, "hi": 8191, "tokens": 2048, "rope": True, "wide": True},
        # rows rotated elsewhere, an odd number of tokens, int32 block table
        {"name": "write mixed 777 rows", "op": "write", "mode": "mixed", "batch": 5, "hkv": 2,
         "lo": 3, "hi": 1001, "tokens": 777, "rope": False, "wide": False},
        # the history that one prefill chunk attends to
        {"name": "read 1 x 2047", "op": "read", "batch": 1, "hkv": 2, "lo": 2047, "hi": 2047,
         "frac": 0.0, "wide": True},
        # the histories of a mixed pass with many decode rows
        {"name": "read 32 x 8191", "op": "read", "batch": 32, "hkv": 2, "lo": 1, "hi": 8191,
         "frac": 0.0, "wide": True},
        # one user, a short context: latency
        {"name": "attend 1 x 511", "op": "attend", "batch": 1, "hkv": 2, "group": 7, "lo": 511,
         "hi": 511, "wide": True},
        # a small ragged batch, an empty row among it
        {"name": "attend 8 x 0-4096", "op": "attend", "batch": 8, "hkv": 2, "group": 7, "lo": 0,
         "hi": 4096, "wide": False},
        # the decode benchmark's batch and context
        {"name": "attend 256 x 4096", "op": "attend", "batch": 256, "hkv": 2, "group": 7,
         "lo": 4096, "hi": 4096, "wide": True},
        # long contexts, ragged
        {"name": "attend 64 x 32768", "op": "attend", "batch": 64, "hkv": 2, "group": 7,
         "lo": 16001, "hi": 32768, "wide": False},
        # one user's token
        {"name": "sample 1", "op": "sample", "rows": 1, "vocab": 151936, "mix": "filtered"},
        # a decode batch, every kind of row in it
        {"name": "sample 64", "op": "sample", "rows": 64, "vocab": 151936, "mix": "all"},
        # a large batch over a smaller, odd vocabulary, no filters
        {"name": "sample 256 x 32003", "op": "sample", "rows": 256, "vocab": 32003,
         "mix": "open"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "write", "read", "attend", "attend", "sample", "sample"])
    wide = rng.random() < 0.5
    if op == "write":
        batch = _log_int(rng, 1, 64)
        mode = rng.choice(["decode", "mixed"])
        tokens = batch if mode == "decode" else max(batch, _log_int(rng, 1, 2048))
        lo = rng.randrange(0, 64)
        return {"op": op, "mode": mode, "batch": batch, "hkv": rng.choice([1, 2, 4]), "lo": lo,
                "hi": lo + _log_int(rng, 1, 8000), "tokens": tokens,
                "rope": rng.random() < 0.5, "wide": wide}
    if op == "read":
        hi = _log_int(rng, 1, 8191)
        return {"op": op, "batch": _log_int(rng, 1, 32), "hkv": rng.choice([1, 2, 4]),
                "lo": rng.randrange(0, hi + 1), "hi": hi, "frac": rng.choice([0.0, 0.37]),
                "wide": wide}
    if op == "attend":
        batch, hkv = _log_int(rng, 1, 256), rng.choice([1, 2, 4])
        hi = _log_int(rng, 1, min(32768, 1500000 // (batch * hkv)))
        return {"op": op, "batch": batch, "hkv": hkv, "group": rng.choice([1, 2, 4, 5, 7, 8]),
                "lo": rng.randrange(0, hi + 1), "hi": hi, "wide": wide}
    return {"op": op, "rows": _log_int(rng, 1, 64), "vocab": _log_int(rng, 17, 151936),
            "mix": rng.choice(["filtered", "all", "open"])}


# ---- lengths and sizes: a function of the case alone ------------------------------


def _spread(lo, hi, n):
    """n whole numbers spread evenly from hi down to lo."""
    return [hi - (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _chunks(case):
    """Tokens of each sequence of a write: one each, or ragged parts of the total
    (single decode rows first, as a scheduler lays a mixed pass out)."""
    n, total = case["batch"], case["tokens"]
    if case["mode"] == "decode" or n == 1:
        return [total // n] * n
    ones = n // 2
    weights = [1 + 3 * i for i in range(n - ones)]
    rest = total - n
    got = [1] * ones + [1 + rest * w // sum(weights) for w in weights]
    got[-1] += total - sum(got)
    return got


def _write_plan(case):
    hist = _spread(case["lo"], case["hi"], case["batch"])
    return hist, _chunks(case)


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 2 * n + 32 * case["rows"], "flops": 3 * n}
    hkv = case["hkv"]
    entry = 8 if case["wide"] else 4
    if case["op"] == "write":
        hist, chunks = _write_plan(case)
        t = sum(chunks)
        hq = 7 * hkv
        pages = sum((h + c - 1) // PAGE - h // PAGE + 1 for h, c in zip(hist, chunks))
        rows = sum(h + c - h // PAGE * PAGE for h, c in zip(hist, chunks))
        rot = t * hq * D * 4 + t * 2 * D * 2 if case["rope"] else 0
        fresh = t * 2 * hkv * D * 3 + pages * (2 * hkv * 4 + entry)
        back = rows * 2 * hkv * D * 3
        return {"bytes": rot + fresh + back, "flops": t * (hq + 2 * hkv) * D * 3}
    lens = _spread(case["lo"], case["hi"], case["batch"])
    if case["op"] == "read":
        starts = [int(n * case["frac"]) for n in lens]
        rows = sum(lens) - sum(starts)
        pages = sum(-(-n // PAGE) - s // PAGE for n, s in zip(lens, starts))
        return {"bytes": rows * 2 * hkv * D * 3 + pages * (2 * hkv * 4 + entry) + 1,
                "flops": rows * 2 * hkv * D}
    hq = hkv * case["group"]
    rows = sum(lens)
    pages = sum(-(-n // PAGE) for n in lens)
    return {"bytes": rows * 2 * hkv * D + pages * (2 * hkv * 4 + entry)
            + case["batch"] * hq * D * 4, "flops": 4 * rows * hq * D}


# ---- inputs ------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _kv_values(shape, g):
    """Rows as a model makes them: unit normal, a few channels several times larger."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    x[..., 3] *= 6
    x[..., 40] *= 3
    return x


def _stored(n_pages, hkv, g):
    """Codes and scales of a pool whose pages hold such rows."""
    k = torch.empty((n_pages, hkv, PAGE, D), dtype=torch.int8, device="cuda")
    v = torch.empty_like(k)
    scales = torch.empty((n_pages, 2, hkv), device="cuda")
    for a in range(0, n_pages, 16384):
        b = min(n_pages, a + 16384)
        for which, pool in ((0, k), (1, v)):
            x = _kv_values((b - a, hkv, PAGE, D), g)
            x *= torch.rand((b - a, hkv, 1, 1), generator=g, device="cuda") + 0.25
            s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / 126)))
            pool[a:b] = torch.round(x / s[..., None, None]).to(torch.int8)
            scales[a:b, which] = s
    return k, v, scales


def _tables(lens, seed, wide):
    """Scattered pages for sequences of these lengths; page 0 and slot 0 are padding."""
    rng = np.random.default_rng(seed)
    need = [-(-n // PAGE) for n in lens]
    n_pages, n_slots = sum(need) + 1, len(lens) + 1
    free = rng.permutation(n_pages - 1) + 1
    slots = rng.permutation(n_slots - 1) + 1
    table = torch.zeros((n_slots, n_pages), dtype=torch.int64 if wide else torch.int32)
    at = 0
    for s, n in zip(slots, need):
        table[s, :n] = torch.from_numpy(free[at:at + n])
        at += n
    return n_pages, n_slots, torch.from_numpy(slots).cuda(), table.cuda()


def _rotary(positions):
    inv = 1.0 / (1e6 ** (torch.arange(0, D, 2, dtype=torch.float64) / D))
    angle = positions.to(torch.float64)[:, None] * inv
    angle = torch.cat((angle, angle), dim=-1)
    return angle.cos().half()[None].cuda(), angle.sin().half()[None].cuda()


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": dict(case)}
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        x = torch.randn((n, v), generator=g, device="cuda") * 2.5 - 2
        top = torch.randint(0, v, (n, min(v, 40)), generator=g, device="cuda")
        x.scatter_add_(1, top, torch.rand(top.shape, generator=g, device="cuda") * 12)
        if v > 1000:
            x[:, v - v // 550:] = -math.inf  # the padded end of the vocabulary
        u = lambda lo, hi: torch.rand(n, generator=g, device="cuda") * (hi - lo) + lo
        pick = lambda p: torch.rand(n, generator=g, device="cuda") < p
        zero = torch.zeros(n, device="cuda")
        temperature, top_k = u(0.3, 1.4), torch.zeros(n, dtype=torch.int64, device="cuda")
        top_p, min_p = zero + 1, zero.clone()
        if case["mix"] != "open":
            some = 1.0 if case["mix"] == "filtered" else 0.5
            ks = torch.tensor([1, 20, 50, 1000], device="cuda")
            k = ks[torch.randint(0, 4, (n,), generator=g, device="cuda")]
            top_k = torch.where(pick(some), k, top_k)
            top_p = torch.where(pick(some), u(0.5, 0.99), top_p)
            min_p = torch.where(pick(some / 2), u(0.001, 0.1), min_p)
            temperature = torch.where(pick((1 - some) / 4), zero, temperature)  # greedy rows
        s.update(logits=x.half(), uniform=u(0, 1).clamp_(max=1 - 2.0 ** -24),
                 temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        return s
    hkv = case["hkv"]
    if case["op"] == "write":
        hist, chunks = _write_plan(case)
        ends = [h + c for h, c in zip(hist, chunks)]
        n_pages, n_slots, slots, table = _tables(ends, seed, case["wide"])
        k, v, scales = _stored(n_pages, hkv, g)
        t = sum(chunks)
        qkv = _kv_values((1, t, 9 * hkv, D), g).reshape(1, t, 9 * hkv * D).half()
        pos = torch.cat([torch.arange(h, e) for h, e in zip(hist, ends)])
        cos, sin = _rotary(pos)
        hist = torch.tensor(hist, device="cuda")
        cu = torch.tensor([0] + np.cumsum(chunks).tolist(), device="cuda")
        lens = torch.zeros(n_slots, dtype=torch.int64, device="cuda")
        lens[slots] = hist
        touched = torch.cat([table[s, h // PAGE:(e - 1) // PAGE + 1].long() for s, h, e in
                             zip(slots.tolist(), hist.tolist(), ends)])
        kn = qkv.view(1, t, 9 * hkv, D)[:, :, 7 * hkv:8 * hkv]
        vn = qkv.view(1, t, 9 * hkv, D)[:, :, 8 * hkv:]
        s.update(k=k, v=v, scales=scales, slots=slots, table=table, qkv=qkv, cos=cos, sin=sin,
                 kv_lens=hist, cu=cu, lens=lens, touched=touched, k_new=kn, v_new=vn,
                 starts=hist // PAGE * PAGE, ends=torch.tensor(ends, device="cuda"),
                 window=max(-(-e // PAGE) for e in ends),
                 k_out=torch.zeros(k.shape, dtype=torch.float16, device="cuda"),
                 v_out=torch.zeros(k.shape, dtype=torch.float16, device="cuda"))
        return s
    lens = _spread(case["lo"], case["hi"], case["batch"])
    n_pages, n_slots, slots, table = _tables(lens, seed, case["wide"])
    k, v, scales = _stored(n_pages, hkv, g)
    ends = torch.tensor(lens, device="cuda")
    s.update(k=k, v=v, scales=scales, slots=slots, table=table, ends=ends,
             window=max(max(-(-n // PAGE) for n in lens), 1))
    if case["op"] == "read":
        s.update(starts=torch.tensor([int(n * case["frac"]) for n in lens], device="cuda"),
                 k_out=torch.zeros(k.shape, dtype=torch.float16, device="cuda"),
                 v_out=torch.zeros(k.shape, dtype=torch.float16, device="cuda"))
    else:
        s["q"] = torch.randn((1, case["batch"], hkv * case["group"], D), generator=g,
                             device="cuda").half()
    return s


# ---- the plain forms ------------------------------------------------------------------


def _rotate(x, cos, sin):
    """Rotary embedding of (T, heads, D) rows in 32 bits."""
    half = torch.cat((-x[..., D // 2:], x[..., :D // 2]), dim=-1)
    return x * cos[:, None] + half * sin[:, None]


def _need(amax):
    """The smallest 2^e with amax <= 127 * 2^e, -24 <= e <= 9."""
    m, e = torch.frexp(amax)
    e = torch.where(m * 128 <= 127, e - 7, e - 6)
    e = torch.where(amax > 0, e, -24).clamp(-24, 9)
    return torch.ldexp(torch.ones_like(amax), e)


def _plain_write(s):
    hkv = s["case"]["hkv"]
    if s["case"]["rope"]:
        rows = s["qkv"][0].float().unflatten(-1, (9 * hkv, D))
        cos, sin = s["cos"][0].float(), s["sin"][0].float()
        q = _rotate(rows[:, :7 * hkv], cos, sin).half()[None]
        k = _rotate(rows[:, 7 * hkv:8 * hkv], cos, sin)
        v = rows[:, 8 * hkv:]
    else:
        q, k, v = None, s["k_new"][0].float(), s["v_new"][0].float()
    t = torch.arange(k.shape[0], device=k.device)
    if s["case"]["mode"] == "decode":
        seq, pos = t, s["lens"][s["slots"]]
    else:
        seq = torch.searchsorted(s["cu"][1:], t, right=True)
        pos = s["kv_lens"][seq] + t - s["cu"][seq]
    page, off = s["table"][s["slots"][seq], pos // PAGE].long(), pos % PAGE
    new = torch.stack((k, v), dim=1)                                # (T, 2, hkv, D)
    n_pages = s["k"].shape[0]
    amax = torch.zeros((n_pages, 2, hkv), device=k.device)
    amax.index_reduce_(0, page, new.abs().amax(-1), "amax")
    first = torch.full((n_pages,), PAGE, device=k.device).scatter_reduce_(0, page, off, "amin")
    at = s["touched"]
    old = torch.where(first[at, None, None] > 0, s["scales"][at], 0)
    scale = torch.maximum(old, _need(amax[at]))
    older = torch.arange(PAGE, device=k.device) < first[at, None]    # (P, PAGE)
    for i, pool in enumerate((s["k"], s["v"])):
        codes = pool[at].float()
        again = torch.round(codes * (old / scale)[:, i, :, None, None])
        pool[at] = torch.where(older[:, None, :, None], again, codes).to(torch.int8)
    s["scales"][at] = scale
    codes = torch.round(new / s["scales"][page][..., None]).clamp(-127, 127).to(torch.int8)
    s["k"][page, :, off] = codes[:, 0]
    s["v"][page, :, off] = codes[:, 1]
    return q


def _plain_read(s):
    pages = s["table"][s["slots"], :s["window"]].long()                # (B, W)
    pos = torch.arange(s["window"] * PAGE, device=pages.device).view(1, -1, PAGE)
    want = (pos >= s["starts"][:, None, None]) & (pos < s["ends"][:, None, None])
    for i, (pool, out) in enumerate(((s["k"], s["k_out"]), (s["v"], s["v_out"]))):
        x = pool[pages].float() * s["scales"][pages][:, :, i, :, None, None]
        out[pages] = torch.where(want[:, :, None, :, None], x.half(), out[pages])


def _plain_attend(s):
    b, hkv, group = s["case"]["batch"], s["case"]["hkv"], s["case"]["group"]
    pages = s["table"][s["slots"], :s["window"]].long()
    rows = s["window"] * PAGE
    seen = torch.arange(rows, device=pages.device) < s["ends"][:, None]  # (B, rows)
    q = s["q"][0].float().view(b, hkv, group, D)
    sc = s["scales"][pages][..., None, None]
    k = (s["k"][pages].float() * sc[:, :, 0]).transpose(1, 2).reshape(b, hkv, rows, D)
    x = (q @ k.transpose(2, 3)) * D ** -0.5
    del k
    x = torch.where(seen[:, None, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.where(seen[:, None, None], torch.exp(x - top), 0)
    total = p.sum(-1, keepdim=True)
    v = (s["v"][pages].float() * sc[:, :, 1]).transpose(1, 2).reshape(b, hkv, rows, D)
    o = (p @ v) / torch.where(total > 0, total, 1)
    return o.reshape(1, b, hkv * group, D).half()


def _plain_sample(s):
    x = s["logits"].double()
    n, v = x.shape
    t = s["temperature"].double()[:, None]
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    top = order.values[:, :1]
    w = torch.exp((order.values - top) / torch.where(t > 0, t, 1))
    rank = torch.arange(v, device=x.device)
    k = s["top_k"][:, None]
    keep = (rank < torch.where((k > 0) & (k < v), k, v)) & (w > 0)
    cum = torch.cumsum(torch.where(keep, w, 0), dim=-1)
    p = s["top_p"].double()[:, None]
    before = torch.cat((torch.zeros_like(cum[:, :1]), cum[:, :-1]), dim=-1)
    keep &= (p >= 1) | (before < p * cum[:, -1:]) | (rank == 0)
    keep &= w >= s["min_p"].double()[:, None]
    keep |= rank == 0
    kept = keep.sum(-1, keepdim=True)
    mass = cum.gather(1, kept - 1)
    at = (cum <= s["uniform"].double()[:, None] * mass).sum(-1, keepdim=True)
    at = torch.minimum(at, kept - 1)
    at = torch.where(t > 0, at, 0)
    return order.indices.gather(1, at)[:, 0]


# ---- one pass -------------------------------------------------------------------------


def run(state):
    s = state
    op = s["case"]["op"]
    if own:
        from custom_inference_engine_b200 import native

        native.load_ops()
        ops = torch.ops.inference
        if op == "sample":
            return ops.sample_rows(s["logits"], s["uniform"], s["temperature"], s["top_k"],
                                   s["top_p"], s["min_p"])
        if op == "attend":
            return ops.gqa_decode_attention_q8(s["q"], s["k"], s["v"], s["scales"], s["ends"],
                                               s["slots"], s["table"])
        q = None
        if op == "write":
            pool = (s["k"], s["v"], s["scales"])
            if s["case"]["mode"] == "decode":
                at = (s["lens"], s["slots"], s["table"])
                if s["case"]["rope"]:
                    q = ops.rope_kv_q8_decode_update(s["qkv"], s["cos"], s["sin"], *pool, *at)
                else:
                    ops.kv_q8_decode_update(*pool, *at, s["k_new"], s["v_new"])
            else:
                at = (s["cu"], s["kv_lens"], s["slots"], s["table"])
                if s["case"]["rope"]:
                    q = ops.rope_kv_q8_mixed_update(s["qkv"], s["cos"], s["sin"], *pool, *at)
                else:
                    ops.kv_q8_mixed_update(*pool, *at, s["k_new"], s["v_new"])
        ops.kv_q8_read(s["k"], s["v"], s["scales"], s["starts"], s["ends"], s["slots"],
                       s["table"], s["k_out"], s["v_out"])
    else:
        if op == "sample":
            return _plain_sample(s)
        if op == "attend":
            return _plain_attend(s)
        q = _plain_write(s) if op == "write" else None
        _plain_read(s)
    out = [s["k_out"], s["v_out"]]
    if op == "write":
        out.append(s["scales"])
        if q is not None:
            out.append(q)
    return out


# ---- the definitions in 64 bits ---------------------------------------------------------


def _exact_rotate(x, angle_cos, angle_sin):
    lo, hi = x[..., :32], x[..., 32:]
    c, n = angle_cos[:, None], angle_sin[:, None]
    return np.concatenate((lo * c[..., :32] - hi * n[..., :32],
                           hi * c[..., 32:] + lo * n[..., 32:]), axis=-1)


def _exact_write(case, s):
    hkv = case["hkv"]
    host = lambda x: x.cpu().numpy()
    codes = [host(s["k"]).astype(np.float64), host(s["v"]).astype(np.float64)]
    scales = host(s["scales"]).astype(np.float64)
    table, slots = host(s["table"]), host(s["slots"])
    rows = host(s["qkv"])[0].astype(np.float64).reshape(-1, 9 * hkv, D)
    q, k, v = rows[:, :7 * hkv], rows[:, 7 * hkv:8 * hkv], rows[:, 8 * hkv:]
    if case["rope"]:
        cos, sin = host(s["cos"])[0].astype(np.float64), host(s["sin"])[0].astype(np.float64)
        q, k = _exact_rotate(q, cos, sin), _exact_rotate(k, cos, sin)
    out = [np.zeros_like(codes[0]), np.zeros_like(codes[1])]
    hist, chunks = _write_plan(case)
    at = 0
    for slot, h, c in zip(slots, hist, chunks):
        for j in range(h // PAGE, (h + c - 1) // PAGE + 1):
            page = table[slot, j]
            a, b = max(h, j * PAGE), min(h + c, (j + 1) * PAGE)
            r0, r1 = a - j * PAGE, b - j * PAGE
            for i, x in enumerate((k, v)):
                x = x[at + a - h:at + b - h]
                for head in range(hkv):
                    most = np.abs(x[:, head]).max()
                    e = -24
                    while e < 9 and most > 127 * 2.0 ** e:
                        e += 1
                    old = scales[page, i, head] if r0 else 0.0
                    scale = max(old, 2.0 ** e)
                    tile = codes[i][page, head]
                    tile[:r0] = np.rint(tile[:r0] * (old / scale))
                    tile[r0:r1] = np.clip(np.rint(x[:, head] / scale), -127, 127)
                    scales[page, i, head] = scale
                    out[i][page, head, :r1] = tile[:r1] * scale
        at += c
    outs = [torch.from_numpy(x) for x in (out[0], out[1], scales)]
    return outs + ([torch.from_numpy(q)[None]] if case["rope"] else [])


def exact(case, seed):
    """The outputs from the definitions, sequence by sequence in 64 bits; sampled
    tokens are whole numbers and have no other value than the plain form's."""
    if case["op"] == "sample":
        return None
    s = prepare(case, seed)
    if case["op"] == "write":
        return _exact_write(case, s)
    lens = _spread(case["lo"], case["hi"], case["batch"])
    slots = s["slots"].tolist()
    if case["op"] == "read":
        outs = []
        for i, pool in ((0, s["k"]), (1, s["v"])):
            out = torch.zeros(pool.shape, dtype=torch.float64, device=pool.device)
            for slot, n in zip(slots, lens):
                for a in range(int(n * case["frac"]) // PAGE * PAGE, n, 4096 * PAGE):
                    pos = torch.arange(max(a, int(n * case["frac"])), min(n, a + 4096 * PAGE),
                                       device=pool.device)
                    page, off = s["table"][slot, pos // PAGE].long(), pos % PAGE
                    out[page, :, off] = pool[page, :, off].double() * \
                        s["scales"][page, i].double()[..., None]
            outs.append(out)
        return outs
    hkv, group = case["hkv"], case["group"]
    o = torch.zeros((1, case["batch"], hkv * group, D), dtype=torch.float64, device="cuda")
    for b, (slot, n) in enumerate(zip(slots, lens)):
        if n == 0:
            continue
        pages = s["table"][slot, :-(-n // PAGE)].long()
        for h in range(hkv):
            scale = s["scales"][pages, :, h].double()
            k = (s["k"][pages, h].double() * scale[:, 0, None, None]).reshape(-1, D)[:n]
            v = (s["v"][pages, h].double() * scale[:, 1, None, None]).reshape(-1, D)[:n]
            x = s["q"][0, b, h * group:(h + 1) * group].double() @ k.T / 8
            o[0, b, h * group:(h + 1) * group] = torch.softmax(x, dim=-1) @ v
    return o
