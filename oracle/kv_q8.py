"""The 8-bit KV pool's definition in float64: page by page quantisation, read
back and decode attention over the codes."""
import math

import torch

PAGE = 16


def rope_fp32(x, cos, sin):
    """x * cos + rotate_half(x) * sin of (1, T, H, D) rows, every operation rounded
    to fp32 (the kernels' recipe; they round the result once more)."""
    x, c, s = x.float(), cos.float().unsqueeze(2), sin.float().unsqueeze(2)
    half = x.shape[-1] // 2
    rot = torch.cat((-x[..., half:], x[..., :half]), dim=-1)
    return x * c + rot * s


def page_scale(amax: float) -> float:
    """The smallest 2^e, -24 <= e <= 9, with amax <= 127 * 2^e (2^9 beyond)."""
    e = -24
    while e < 9 and amax > 127 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def write_page(codes, scale, off, rows):
    """Rows (n, D) into a page's codes (PAGE, D) float64 from row ``off`` on; returns
    the page's new scale."""
    rows = torch.nan_to_num(rows.double(), nan=0.0, posinf=math.inf, neginf=-math.inf)
    old = scale if off > 0 else 0.0
    new = max(old, page_scale(rows.abs().max().item()))
    codes[:off] = torch.round(codes[:off] * (old / new))
    codes[off:off + rows.shape[0]] = torch.round(rows / new).clamp(-127, 127)
    return new


def update(k, v, scales, chunks, block_table, k_new, v_new):
    """``chunks``: (slot, first position, first row of k_new, rows), in place. k, v
    (n_pages, H, PAGE, D) int8, scales (n_pages, 2, H) fp32; new rows (T, H, D)."""
    for slot, start, row0, n in chunks:
        pos = start
        while pos < start + n:
            off = pos % PAGE
            take = min(PAGE - off, start + n - pos)
            page = int(block_table[slot, pos // PAGE])
            at = row0 + pos - start
            for i, (pool, new) in enumerate(((k, k_new), (v, v_new))):
                for h in range(pool.shape[1]):
                    codes = pool[page, h].double()
                    s = write_page(codes, float(scales[page, i, h]), off, new[at:at + take, h])
                    pool[page, h] = codes.to(torch.int8)
                    scales[page, i, h] = s
            pos += take


def read(k, v, scales, starts, lens, slot_ids, block_table, k_out, v_out):
    for slot, a, z in zip(slot_ids.tolist(), starts.tolist(), lens.tolist()):
        for pos in range(a, z):
            page, off = int(block_table[slot, pos // PAGE]), pos % PAGE
            k_out[page, :, off] = (k[page, :, off].double()
                                   * scales[page, 0].double()[:, None]).half()
            v_out[page, :, off] = (v[page, :, off].double()
                                   * scales[page, 1].double()[:, None]).half()


def decode_attention(q, k, v, scales, lens, slot_ids, block_table):
    """softmax(q k^T / sqrt(D)) v in float64 over code * scale, with a bound on what
    the kernel's own arithmetic may differ by (see ``tests/test_kv_q8_gpu.py``)."""
    _, B, hq, D = q.shape
    hkv = k.shape[1]
    group = hq // hkv
    o = torch.zeros(B, hq, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(o)
    for b in range(B):
        n = int(lens[b])
        if n == 0:
            continue
        pages = block_table[slot_ids[b], :-(-n // PAGE)].long()
        for h in range(hkv):
            sc = scales[pages, :, h].double()
            kk = (k[pages, h].double() * sc[:, 0, None, None]).reshape(-1, D)[:n]
            vv = (v[pages, h].double() * sc[:, 1, None, None]).reshape(-1, D)[:n]
            qq = q[0, b, h * group:(h + 1) * group].double()
            s = qq @ kk.T / math.sqrt(D)
            p = torch.exp(s - s.max(-1, keepdim=True).values)
            total = p.sum(-1, keepdim=True)
            out = p @ vv / total
            o[b, h * group:(h + 1) * group] = out
            # e: error of a score, from D fp32 additions (each at most 2^-23 of the
            # running sum of magnitudes, tensor cores may truncate), the scaling, and
            # the subtraction of the maximum and multiplication by log2(e)
            e = (qq.abs() @ kk.abs().T / math.sqrt(D)).amax(-1, keepdim=True) * (D + 2) * 2.0 ** -23
            e = e + (s.max(-1, keepdim=True).values - s.min(-1, keepdim=True).values) * 2.0 ** -22
            mean = p @ vv.abs() / total
            # p's rounding to fp16 (half a step, 2^-11, or half the smallest subnormal,
            # 2^-25), exp2's error 2^-22, the score error in numerator and denominator,
            # sums of n terms in fp32 merged over warps and splits, one fp16 rounding
            sums = (n + 64) * 2.0 ** -23
            tol[b, h * group:(h + 1) * group] = (
                2.0 ** -11 * out.abs() + (2.0 ** -11 + 2 * e.expm1() + 2.0 ** -20 + 2 * sums) * mean
                + 2.0 ** -25 * vv.abs().sum(0) / total + 2.0 ** -25)
    return o[None], tol[None]
