"""Plain implementations of the paged-cache operators on the CPU: requests one
after the other, numbers in 64 bits."""
import math

import numpy as np
import torch


def plan(q_len, kv_len, table, free, state, page, n_tok):
    """What khq_paged_plan writes, from lists; table and free are changed copies."""
    table = [list(r) for r in table]
    free, n_pages, width = list(free), len(free), len(table[0])
    head, count = state
    cu, kv_out, seq_kv, positions, slots, refused = [0], [], [], [], [], 0
    rows = taken = wanted = 0
    back = []
    for s, (q, kv) in enumerate(zip(q_len, kv_len)):
        has = -(-kv // page)
        rows += max(q, 0)
        cu.append(min(rows, n_tok))
        if q <= 0:
            if q < 0:
                back += table[s][:has]
            kv_out.append(0 if q < 0 else kv)
            seq_kv.append(kv_out[-1])
            continue
        want = -(-(kv + q) // page)
        ok = want <= width and rows <= n_tok
        if ok:
            wanted += want - has
            ok = want == has or wanted <= count
        if ok:
            for p in range(has, want):
                table[s][p] = free[(head + taken) % n_pages]
                taken += 1
        kv_out.append(kv + q if ok else kv)
        seq_kv.append(kv + q if ok else 0)
        refused += not ok
        for i in range(cu[-1] - cu[-2]):
            pos = kv + i
            positions.append(pos)
            entry = table[s][pos // page] if ok else -1
            slots.append(entry * page + pos % page if 0 <= entry < n_pages else -1)
    for j, p in enumerate(back):
        free[(head + count + j) % n_pages] = p
    pad = n_tok - len(slots)
    return {"table": table, "free": free, "cu_q": cu, "seq_kv": seq_kv, "kv_out": kv_out,
            "state_out": [(head + taken) % n_pages, count - taken + len(back)],
            "status": [refused], "positions": positions + [0] * pad, "slots": slots + [-1] * pad}


def norm_rope(x, w, positions, eps, theta, rot, round_to=None):
    """[n][H][D] in 64 bits: (normed, rotated, a bound of the pair's size)."""
    x = x.detach().cpu().double()
    d = x.shape[-1]
    y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + eps)
    if w is not None:
        y = y * w.detach().cpu().double()
    z = y.to(round_to).double() if round_to is not None else y
    out = z.clone()
    half = rot // 2
    size = z.abs().clone()
    if rot:
        f = theta ** (-2.0 * torch.arange(half, dtype=torch.float64) / rot)
        ang = positions.detach().cpu().double()[:, None, None] * f
        a, b = z[..., :half], z[..., half:rot]
        out[..., :half] = a * torch.cos(ang) - b * torch.sin(ang)
        out[..., half:rot] = a * torch.sin(ang) + b * torch.cos(ang)
        size[..., :half] = size[..., half:rot] = a.abs() + b.abs()
    return y, out, size


def gather(pages, row, n, page):
    """The first n tokens of a block table's row: [n][H][D] in 64 bits."""
    pages = pages.detach().cpu()
    t = torch.arange(n)
    return pages[row.long()[t // page], t % page].double()


def attn(q, k_pages, v_pages, cu_q, seq_kv, table, scale, gate=None):
    """(out, bound) in 64 bits, [n][H_q][D]: the attention and, for tolerances,
    sum of w |v| with the largest error of a score in it.  Rows of no sequence
    are NaN in out."""
    n, hq, d = q.shape
    page, hkv = k_pages.shape[1], k_pages.shape[2]
    qc, cu, kv, tab = q.detach().cpu().double(), cu_q.tolist(), seq_kv.tolist(), table.cpu()
    out = torch.full((n, hq, d), math.nan, dtype=torch.float64)
    bound = torch.zeros((n, hq, d), dtype=torch.float64)
    half = torch.finfo(q.dtype).eps / 2
    for s in range(len(kv)):
        a, b = cu[s], cu[s + 1]
        if a == b:
            continue
        nk = kv[s]
        k, v = gather(k_pages, tab[s], nk, page), gather(v_pages, tab[s], nk, page)
        for i in range(a, b):
            vis = nk - (b - a) + (i - a) + 1
            if vis <= 0:
                out[i] = 0
                continue
            kk = k[:vis].repeat_interleave(hq // hkv, 1)
            vv = v[:vis].repeat_interleave(hq // hkv, 1)
            sc = torch.einsum("hd,thd->ht", qc[i], kk) * scale
            w = torch.softmax(sc, 1)
            out[i] = torch.einsum("ht,thd->hd", w, vv)
            mass = torch.einsum("ht,thd->hd", w, vv.abs())
            # a score's error: d + 2 roundings of 2^-24 of sum |q k|, and of the
            # score itself in the exponent's argument (three)
            err = (d + 2) * 2.0 ** -24 * torch.einsum("hd,thd->ht", qc[i].abs(), kk.abs()).amax(1) * abs(scale)
            err = err + 3 * 2.0 ** -24 * (sc.abs().amax(1) + 1) * 1.5
            # weights: that, their rounding to the type, the exponential's (2^-22), sums
            # in 32 bits (vis roundings at worst); numerator and denominator
            bound[i] = 2 * (half + err + 2.0 ** -22 + vis * 2.0 ** -24)[:, None] * mass
    if gate is not None:
        g = torch.sigmoid(gate.detach().cpu().double())
        out, bound = out * g, bound * g + 2.0 ** -20 * out.abs().nan_to_num()
    return out, bound


def rand_cache(n_seq, kv, page, hkv, d, dtype, seed, device="cpu", extra=3, fill=None):
    """Pages of n_seq sequences in no order, and their block table.  fill: what
    the slots of no token hold."""
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // page) for n in kv]
    n_pages, width = sum(held) + extra, max(max(held), 1) + 1
    k = torch.randn((n_pages, page, hkv, d), generator=g).to(dtype)
    v = torch.randn((n_pages, page, hkv, d), generator=g).to(dtype)
    order, at = rng.permutation(n_pages), 0
    table = torch.zeros((n_seq, width), dtype=torch.int32)
    if fill is not None:
        keep = torch.zeros((n_pages, page), dtype=torch.bool)
    for s, n in enumerate(held):
        table[s, :n] = torch.from_numpy(order[at: at + n].astype(np.int32))
        table[s, n:] = 1 << 30  # never looked at
        if fill is not None:
            t = torch.arange(kv[s])
            keep[table[s].long()[t // page], t % page] = True
        at += n
    if fill is not None:
        k[~keep], v[~keep] = fill, fill
    return k.to(device), v.to(device), table.to(device)
