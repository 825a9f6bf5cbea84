"""The paged cache's operators against plain implementations in 64 bits
(tests/pagedref.py)."""
import math
import threading

import numpy as np
import pytest
import torch

import pagedref
from khq import paged

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def say(*a):
    print(*a, flush=True)


def i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


# ---------------------------------------------------------------------- plan
def plan_state(n_seq, page, width, n_pages, q, kv, seed, device, head=None):
    rng = np.random.default_rng(seed)
    order, at = rng.permutation(n_pages).tolist(), 0
    table = rng.integers(0, n_pages, (n_seq, width)).tolist()
    for s in range(n_seq):
        for p in range(min(-(-kv[s] // page), width)):
            table[s][p] = order[at]
            at += 1
    head = n_pages // 3 if head is None else head
    count = n_pages - at
    free = [0] * n_pages
    for j in range(count):
        free[(head + j) % n_pages] = order[at + j]
    return table, free, [head, count]


def run_plan(q, kv, table, free, state, page, n_tok, device, in_place=False):
    n = len(q)
    t = dict(q=i32(q, device), kv=i32(kv, device), table=i32(table, device), free=i32(free, device),
             state=i32(state, device))
    z = lambda *s: torch.full(s, -77, dtype=torch.int32, device=device)  # noqa: E731
    o = dict(cu_q=z(n + 1), seq_kv=z(n), kv_out=t["kv"] if in_place else z(n),
             state_out=t["state"] if in_place else z(2), status=z(1), positions=z(n_tok),
             slots=z(n_tok))
    paged.plan(t["q"], t["kv"], t["table"], t["free"], t["state"], page_size=page, **o)
    return {k: v.tolist() for k, v in o.items()} | {"table": t["table"].tolist(),
                                                    "free": t["free"].tolist()}


def check_plan(q, kv, page, width, n_pages, n_tok, device, seed=0, head=None):
    table, free, state = plan_state(len(q), page, width, n_pages, q, kv, seed, device, head)
    want = pagedref.plan(q, kv, table, free, state, page, n_tok)
    for in_place in (False, True):
        got = run_plan(q, kv, table, free, state, page, n_tok, device, in_place)
        for name in want:
            assert got[name] == want[name], name
    return want


@pytest.mark.parametrize("n_seq,page,q_hi,seed", [
    (1, 16, 1, 1), (1, 1, 5, 2), (64, 16, 1, 3), (63, 48, 9, 4), (300, 7, 20, 5), (1025, 16, 2, 6),
    (4096, 64, 3, 7), (700, 128, 150, 8)])
def test_plan(n_seq, page, q_hi, seed, device):
    rng = np.random.default_rng(seed)
    q = rng.integers(1, q_hi + 1, n_seq)
    q[rng.random(n_seq) < 0.2] = 0
    q[rng.random(n_seq) < 0.1] = -1
    kv = rng.integers(0, 6 * page, n_seq)
    kv[rng.random(n_seq) < 0.1] = 0
    q, kv = q.tolist(), kv.tolist()
    pages = sum(-(-(max(a, 0) + b) // page) for a, b in zip(q, kv)) + 3
    say("plan", n_seq, page, q_hi)
    w = check_plan(q, kv, page, 8 + q_hi // page, pages, sum(max(0, a) for a in q) + 11, device, seed)
    assert w["status"] == [0]


def test_plan_refusals(device):
    # too few pages: the second request waits, the third needs none, the last is refused
    # with it though its own would be there
    w = check_plan([3, 40, 1, 2], [14, 0, 1, 16], 16, 8, 6, 50, device)
    assert w["status"] == [2] and w["slots"][3:43] == [-1] * 40 and w["seq_kv"] == [17, 0, 2, 0]
    # a table too narrow, a batch too short; the others go on
    w = check_plan([1, 1, 1], [32, 5, 6], 16, 2, 9, 3, device)
    assert w["status"] == [1] and w["seq_kv"] == [0, 6, 7]
    w = check_plan([4, 4, -1, 2], [4, 5, 6, 1], 16, 2, 9, 9, device)
    assert w["status"] == [1] and w["cu_q"] == [0, 4, 8, 8, 9] and w["slots"][8] == -1
    # no free page at all, none needed; nothing to do; everything ended
    check_plan([1, 1], [3, 4], 16, 1, 2, 2, device)
    check_plan([0, 0], [3, 0], 16, 1, 2, 0, device)
    w = check_plan([-1, -5, -1], [40, 0, 16], 16, 4, 4, 2, device, head=3)
    assert w["state_out"] == [3, 4]
    # lengths that pass 32 bits
    big = 2 ** 31 - 1
    w = check_plan([big, big, 1, big], [0, 0, 3, 7], 16, 8, 9, 4, device)
    assert w["status"] == [4]


def test_plan_bad_entries(device):
    """Entries outside the cache give slot -1; a state outside its range is taken into it."""
    w = check_plan([2, 2], [3, 3], 4, 3, 4, 4, device)
    assert min(w["slots"]) >= 0
    t = [[99, 0, 0], [0, -5, 0]]
    got = run_plan([2, 2], [3, 3], t, [1, -7, 2, 3], [1, 3], 4, 4, device)
    assert got["slots"] == [-1, -1, 3, 8]
    got = run_plan([2, 2], [3, 3], t, [1, 0, 2, 3], [-3, 99], 4, 4, device)
    assert got["state_out"][0] in range(4) and got["state_out"][1] <= 4


def test_page_table_over_many_steps(device):
    """Requests come, grow, end and come again: no page is in two hands, none is lost."""
    rng = np.random.default_rng(5)
    n_seq, page, n_pages = 13, 4, 40
    t = paged.PageTable(n_seq, 12, n_pages, page, 64, device)
    kv = [0] * n_seq
    for step in range(60):
        q = [int(rng.choice([-1, 0, 1, 1, 1, 3, 9])) for _ in kv]
        before = {k: getattr(t, k).tolist() for k in ("table", "free_pages", "state")}
        w = pagedref.plan(q, kv, before["table"], before["free_pages"], before["state"], page, 64)
        t.step(i32(q, device))
        for name, x in (("table", t.table), ("free", t.free_pages), ("cu_q", t.cu_q),
                        ("seq_kv", t.seq_kv), ("kv_out", t.kv_len), ("state_out", t.state),
                        ("status", t.status), ("positions", t.positions), ("slots", t.slots)):
            assert x.tolist() == w[name], (step, name)
        kv = w["kv_out"]
        held = [p for s in range(n_seq) for p in w["table"][s][: -(-kv[s] // page)]]
        free = [w["free"][(w["state_out"][0] + j) % n_pages] for j in range(w["state_out"][1])]
        assert sorted(held + free) == list(range(n_pages))


def test_plan_replayed(device):
    """A captured step follows the lengths it finds, batches of one block and of several."""
    for n_tok in (64, 9000):
        t = paged.PageTable(8, 600, 3000, 16, n_tok, device)
        q = i32([1, 2, 0, 3, 1, 1, 700, 5], device)
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            t.step(q)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            t.step(q)
        for k in range(5):
            ql = [k, 1, 2 * k, -1 if k == 3 else 1, 0, n_tok // 40, 3, 1]
            q.copy_(i32(ql, device))
            s = {n: getattr(t, n).tolist() for n in ("kv_len", "table", "free_pages", "state")}
            w = pagedref.plan(ql, s["kv_len"], s["table"], s["free_pages"], s["state"], 16, n_tok)
            graph.replay()
            torch.cuda.synchronize()
            for name, x in (("table", t.table), ("free", t.free_pages), ("kv_out", t.kv_len),
                            ("state_out", t.state), ("slots", t.slots), ("positions", t.positions)):
                assert x.tolist() == w[name], (k, name)


# ---------------------------------------------------------------------- rows
def check_rows(got, want, size, dtype, normed_step=False):
    """Half a step of the type, and 2^-18 of the pair (the sine and cosine of the hardware,
    32-bit arithmetic); with values rounded before the rotation, half a step of the pair too."""
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps  # a subnormal's step
    tol = half * want.abs() + (2.0 ** -18 + (half if normed_step else 0)) * size + tiny
    err = (got.detach().cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def rows_case(n, hq, hkv, d, rot, dtype, seed, device, pos_hi=100000, weights=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    return dict(q=(2 * r(n, hq, d)).to(dtype).to(device), k=(3 * r(n, hkv, d)).to(dtype).to(device),
                v=r(n, hkv, d).to(dtype).to(device),
                qw=(1 + 0.3 * r(d)).to(device) if weights else None,
                kw=(1 + 0.3 * r(d)).to(device) if weights else None,
                pos=torch.randint(0, pos_hi, (n,), generator=g, dtype=torch.int32).to(device))


@pytest.mark.parametrize("n,hq,hkv,d,rot,dtype", [
    (1, 24, 4, 256, 64, F16), (7, 24, 4, 256, 64, BF16), (33, 32, 8, 128, 128, BF16),
    (5, 8, 8, 64, 64, F16), (3, 5, 1, 64, 16, F16), (9, 3, 3, 128, 48, F16), (2, 40, 2, 256, 256, BF16),
    (300, 24, 4, 256, 64, F16), (4, 6, 2, 128, 0, F16), (70, 1, 1, 64, 32, BF16)])
@pytest.mark.parametrize("weights", [True, False])
def test_rows(n, hq, hkv, d, rot, dtype, weights, device):
    say("rows", n, hq, hkv, d, rot, dtype)
    c = rows_case(n, hq, hkv, d, rot, dtype, n + d, device, weights=weights)
    page, n_pages = 5, n // 3 + 2
    g = torch.Generator().manual_seed(1)
    kp = torch.randn((n_pages, page, hkv, d), generator=g).to(dtype).to(device)
    vp = torch.randn((n_pages, page, hkv, d), generator=g).to(dtype).to(device)
    slots = torch.randperm(n_pages * page, generator=g)[:n].int()
    slots[::4] = -1  # a padded batch's
    if n > 5:
        slots[5] = n_pages * page  # outside the cache
    q_out, k_out, k_n = torch.zeros_like(c["q"]), torch.zeros_like(c["k"]), torch.zeros_like(c["k"])
    want_k, want_v = kp.cpu().clone(), vp.cpu().clone()
    paged.qk_norm_rope(c["q"], c["k"], q_out, positions=c["pos"], q_weight=c["qw"], k_weight=c["kw"],
                       eps=1e-6, theta=1e7, rotary_dim=rot, k_out=k_out, k_normed=k_n, v=c["v"],
                       k_pages=kp, v_pages=vp, slots=slots.to(device))
    _, q_ref, q_size = pagedref.norm_rope(c["q"], c["qw"], c["pos"], 1e-6, 1e7, rot)
    y, k_ref, k_size = pagedref.norm_rope(c["k"], c["kw"], c["pos"], 1e-6, 1e7, rot)
    check_rows(q_out, q_ref, q_size, dtype)
    check_rows(k_out, k_ref, k_size, dtype)
    check_rows(k_n, y, y.abs(), dtype)
    # the cache: the rotated keys and the values at their slots, the rest as it was
    ok = (slots >= 0) & (slots < n_pages * page)
    want_k.view(-1, hkv, d)[slots[ok].long()] = k_out.cpu()[ok]
    want_v.view(-1, hkv, d)[slots[ok].long()] = c["v"].cpu()[ok]
    assert torch.equal(kp.cpu(), want_k) and torch.equal(vp.cpu(), want_v)


def test_rows_strided_in_place(device):
    """One projection's row holds queries, gates, keys and values; the queries become the
    rotated ones, the gates stay; pages are [pages][heads][tokens][dims] of one tensor."""
    for dtype, off in ((F16, 0), (BF16, 3)):  # off: rows at no 16-byte boundary
        n, hq, hkv, d = 19, 6, 2, 128
        g = torch.Generator().manual_seed(3)
        flat = torch.randn(n * 2053 + 8, generator=g).to(dtype).to(device)
        buf = flat[off: off + n * 2053].view(n, 2053)
        before = buf.clone()
        q_gate = buf[:, : 2 * hq * d].unflatten(1, (hq, 2 * d))
        k = buf[:, 2 * hq * d: 2 * hq * d + hkv * d].unflatten(1, (hkv, d))
        v = buf[:, 2 * hq * d + hkv * d: 2 * hq * d + 2 * hkv * d].unflatten(1, (hkv, d))
        both = torch.zeros((4, 2, hkv, 8, d), dtype=dtype, device=device)
        kp, vp = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
        slots = torch.arange(n, dtype=torch.int32, device=device) + 5
        k0 = k.clone()
        paged.qk_norm_rope(q_gate[..., :d], k, q_gate[..., :d], pos0=11, rotary_dim=64, k_out=k, v=v,
                           k_pages=kp, v_pages=vp, slots=slots)
        pos = torch.arange(11, 11 + n)
        old = before[:, : 2 * hq * d].unflatten(1, (hq, 2 * d))
        _, ref, size = pagedref.norm_rope(old[..., :d], None, pos, 1e-6, 1e7, 64)
        check_rows(q_gate[..., :d], ref, size, dtype)
        assert torch.equal(q_gate[..., d:], old[..., d:])
        _, ref, size = pagedref.norm_rope(k0, None, pos, 1e-6, 1e7, 64)
        check_rows(k, ref, size, dtype)
        assert torch.equal(buf[:, -1], before[:, -1])
        flat_k = kp.reshape(-1, hkv, d)
        assert torch.equal(flat_k[5: 5 + n], k) and torch.equal(vp.reshape(-1, hkv, d)[5: 5 + n], v)
        assert not flat_k[:5].any() and not flat_k[5 + n:].any()


def test_rows_edges(device):
    # zeros stay zeros, an infinity's head is what the formula says, its neighbours untouched
    q = torch.randn((2, 3, 64), device=device).to(F16)
    q[0, 0] = 0
    q[1, 1, 5] = math.inf
    out = torch.full_like(q, 7)
    paged.qk_norm_rope(q, None, out, rotary_dim=64, pos0=3)
    assert not out[0, 0].any() and bool(out[1, 1].isnan().any())
    assert bool(out[0, 1:].isfinite().all() and out[1, 0].isfinite().all() and out[1, 2].isfinite().all())
    # far positions: angles in 64 bits
    c = rows_case(40, 2, 2, 128, 128, F16, 5, device, pos_hi=2 ** 31 - 1)
    out = torch.zeros_like(c["q"])
    paged.qk_norm_rope(c["q"], None, out, positions=c["pos"], q_weight=c["qw"], theta=1e4, rotary_dim=128)
    _, ref, size = pagedref.norm_rope(c["q"], c["qw"], c["pos"], 1e-6, 1e4, 128)
    check_rows(out, ref, size, F16)
    # rounded before the rotation, keys alone, no rows
    k_out = torch.zeros_like(c["k"])
    paged.qk_norm_rope(None, c["k"], None, positions=c["pos"], rotary_dim=64, k_out=k_out, round_norm=True)
    _, ref, size = pagedref.norm_rope(c["k"], None, c["pos"], 1e-6, 1e7, 64, round_to=F16)
    check_rows(k_out, ref, size, F16, normed_step=True)
    paged.qk_norm_rope(c["q"][:0], None, out[:0], rotary_dim=64)


# ---------------------------------------------------------------------- attn
@pytest.fixture(params=["tight", "wide"])
def table_width(request, monkeypatch):
    """Tables that hold just the longest sequence, and tables of 2^22 tokens: what they could
    hold decides how many rows are taken at once."""
    if request.param == "wide":
        def wide_case(*args, case=attn_case, **kw):
            c = case(*args, **kw)
            more = (1 << 22) // c["kp"].shape[1] - c["table"].shape[1]
            return dict(c, table=torch.nn.functional.pad(c["table"], (0, more), value=-1))

        monkeypatch.setitem(globals(), "attn_case", wide_case)


def attn_case(lens, hq, hkv, d, page, dtype, seed, device, gate=False, fill=None, pad=0):
    q_len, kv = [a for a, _ in lens], [b for _, b in lens]
    kp, vp, table = pagedref.rand_cache(len(lens), kv, page, hkv, d, dtype, seed, device, fill=fill)
    g = torch.Generator().manual_seed(seed + 1)
    n = sum(q_len) + pad
    qg = (1.5 * torch.randn((n, hq, 2 * d), generator=g)).to(dtype).to(device)
    cu = [0]
    for a in q_len:
        cu.append(cu[-1] + a)
    return dict(q=qg[..., :d], gate=qg[..., d:] if gate else None, kp=kp, vp=vp, table=table,
                cu=i32(cu, device), kv=i32(kv, device), scale=d ** -0.5, max_q=max(max(q_len), 1),
                rows=cu[-1])


def run_attn(c, out=None, **over):
    out = torch.full_like(c["q"], 7, memory_format=torch.contiguous_format) if out is None else out
    kw = dict(cu_q=c["cu"], seq_kv=c["kv"], table=c["table"], max_q=c["max_q"], scale=c["scale"],
              gate=c["gate"])
    kw.update(over)
    paged.attn(c["q"], c["kp"], c["vp"], out, **kw)
    return out


def check_attn(c, out, ref=None):
    want, bound = ref or pagedref.attn(c["q"], c["kp"], c["vp"], c["cu"], c["kv"], c["table"], c["scale"],
                                       c["gate"])
    got = out.detach().cpu().double()
    rows = c["rows"]
    assert bool((got[rows:] == 7).all())  # rows of no sequence: left as they were
    got, want, bound = got[:rows], want[:rows], bound[:rows]
    fine = want.isfinite()
    assert torch.equal(got[~fine].nan_to_num(nan=5), want[~fine].nan_to_num(nan=5))
    half = torch.finfo(out.dtype).eps / 2
    tiny = torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
    tol = half * want.abs() + bound + tiny
    err = (got - want).abs()
    ok = (err <= tol) | ~fine
    assert bool(ok.all()), float((err / tol)[fine].max())


WIDE, COMMON, SMALL = (24, 4, 256), (32, 8, 128), (8, 8, 64)
DECODE = [(1, 1), (1, 17), (1, 700), (1, 64), (1, 333), (1, 2)]
CHUNKS = [(5, 5), (1, 90), (37, 200), (0, 40), (64, 64), (3, 3), (130, 131), (2, 600), (0, 0)]


@pytest.mark.parametrize("heads,page,dtype,lens,gate", [
    (WIDE, 16, F16, DECODE, True), (WIDE, 64, BF16, DECODE, False), (COMMON, 48, BF16, DECODE, True),
    (SMALL, 1, F16, DECODE, False), ((6, 1, 64), 7, BF16, DECODE, True),
    ((40, 2, 128), 128, F16, DECODE, False), ((7, 1, 256), 33, F16, DECODE, False),
    (WIDE, 64, F16, CHUNKS, True), (WIDE, 48, BF16, CHUNKS, False), (COMMON, 16, F16, CHUNKS, True),
    (COMMON, 100, BF16, CHUNKS, False), (SMALL, 7, F16, CHUNKS, True), (SMALL, 256, BF16, CHUNKS, False),
    ((5, 1, 128), 64, F16, CHUNKS, False), ((34, 2, 64), 64, BF16, CHUNKS, True),
    ((3, 3, 256), 1, F16, CHUNKS, False), (WIDE, 64, F16, [(1, 1)], True),
    (WIDE, 16, BF16, [(1, 4500)], False), ((16, 1, 256), 64, F16, [(2, 1025), (4, 90)], True),
    (COMMON, 64, F16, [(256, 1300)], False), (WIDE, 32, F16, [(300, 300)], False)])
@pytest.mark.usefixtures("table_width")
def test_attn(heads, page, dtype, lens, gate, device):
    say("attn", heads, page, dtype, lens, gate)
    c = attn_case(lens, *heads, page, dtype, 11, device, gate=gate, fill=math.nan, pad=3)
    out = run_attn(c)
    check_attn(c, out)
    for _ in range(2):
        assert torch.equal(run_attn(c), out)


@pytest.mark.parametrize("heads,dtype", [(WIDE, F16), (COMMON, BF16), (SMALL, F16)])
@pytest.mark.usefixtures("table_width")
def test_attn_rows_that_see_nothing(heads, dtype, device):
    """More rows than tokens, no tokens at all, lengths below zero."""
    lens = [(6, 2), (4, 0), (40, 33), (1, 0), (1, 5), (300, 20)]
    c = attn_case(lens, *heads, 16, dtype, 3, device, gate=True, fill=math.nan)
    out = run_attn(c)
    check_attn(c, out)
    assert not out[:4].any() and not out[6:10].any()
    c["kv"][1] = -7
    assert torch.equal(run_attn(c), out)


@pytest.mark.parametrize("heads,dtype,lens", [
    (WIDE, F16, [(5, 60), (2, 2)]), (WIDE, F16, [(70, 100)]), (COMMON, BF16, [(3, 40), (4, 4)]),
    (COMMON, F16, [(90, 90), (1, 50)]), (SMALL, BF16, [(9, 77)]), ((2, 2, 64), F16, [(200, 233)])])
@pytest.mark.usefixtures("table_width")
def test_attn_nonfinite_in_masked_places(heads, dtype, lens, device):
    """A new token's infinities and NaN reach the rows that see it, and no other."""
    c = attn_case(lens, *heads, 16, dtype, 21, device)
    page, d = 16, heads[2]
    want, bound = pagedref.attn(c["q"], c["kp"], c["vp"], c["cu"], c["kv"], c["table"], c["scale"])
    cu = c["cu"].tolist()
    for s, (a, kv) in enumerate(lens):
        if a < 2:
            continue
        bad = kv - a + a // 2  # rows a // 2 .. see it
        at = int(c["table"][s, bad // page]), bad % page
        c["vp"][at[0], at[1], :, 1] = math.inf
        c["vp"][at[0], at[1], :, d - 2] = -math.inf
        c["vp"][at[0], at[1], :, d // 2] = math.nan
        last = kv - 1  # and the last row alone sees a key that is not a number
        c["kp"][int(c["table"][s, last // page]), last % page] = math.nan
        want[cu[s] + a // 2: cu[s + 1], :, 1] = math.inf
        want[cu[s] + a // 2: cu[s + 1], :, d - 2] = -math.inf
        want[cu[s] + a // 2: cu[s + 1], :, d // 2] = math.nan
        want[cu[s + 1] - 1] = math.nan
    check_attn(c, run_attn(c), (want, bound))


@pytest.mark.usefixtures("table_width")
def test_attn_large_scores_and_lowest_values(device):
    """Scores far apart, keys of the type's largest values, a mask's lowest value as key."""
    for heads, lens in ((WIDE, [(1, 300), (4, 50)]), (COMMON, [(90, 200)])):
        c = attn_case(lens, *heads, 16, F16, 4, device)
        c["kp"].mul_(8)
        c["q"].mul_(8)  # scores of some hundreds
        out = run_attn(c)
        check_attn(c, out)
        c["scale"] = -c["scale"]
        check_attn(c, run_attn(c))
        c["scale"] = 0.0
        check_attn(c, run_attn(c))
    c = attn_case([(1, 40), (33, 60)], 4, 4, 64, 8, F16, 5, device)
    c["q"][:] = 1
    c["kp"][:] = -65504.0  # every score the same, -4.2e6 * scale
    c["scale"] = 1.0
    out = run_attn(c)
    assert bool(out.isfinite().all())
    check_attn(c, out)


@pytest.mark.usefixtures("table_width")
def test_attn_strides_and_alignment(device):
    """Pages as [pages][heads][tokens][dims] of one tensor, queries at odd addresses and
    strides, heads before tokens, an output of other strides."""
    for heads, lens in ((WIDE, [(1, 70), (1, 9)]), (COMMON, [(40, 90), (3, 17)])):
        hq, hkv, d = heads
        c = attn_case(lens, *heads, 16, F16, 8, device, gate=True)
        want = run_attn(c)
        n_pages = c["kp"].shape[0]
        both = torch.zeros((n_pages, 2, hkv, 16, d), dtype=F16, device=device)
        both[:, 0], both[:, 1] = c["kp"].transpose(1, 2), c["vp"].transpose(1, 2)
        n = c["q"].shape[0]
        odd = torch.zeros(n * (hq * d + 5) + 3, dtype=F16, device=device)[3:].view(n, -1)
        odd[:, : hq * d].view(n, hq, d).copy_(c["q"])
        gate_t = torch.zeros((hq, n, d), dtype=F16, device=device)
        gate_t.copy_(c["gate"].transpose(0, 1))
        out_t = torch.zeros((hq, n, d + 1), dtype=F16, device=device)[..., 1:]
        o = dict(c, q=odd[:, : hq * d].view(n, hq, d), gate=gate_t.transpose(0, 1),
                 kp=both[:, 0].transpose(1, 2), vp=both[:, 1].transpose(1, 2))
        got = run_attn(o, out=out_t.transpose(0, 1))
        assert torch.equal(got, want)


@pytest.mark.parametrize("n,heads", [(900, 128), (1100, 128), (1536, 128), (1100, 256)])
def test_attn_rounds_of_blocks(n, heads, device):
    """A lone prompt of two, three, three full and five rounds of blocks (tiles of 128 rows,
    512 at once): every row tile is some block's.  Checked for four of the heads."""
    c = attn_case([(n, n)], heads, heads, 64, 64, F16, 12, device)
    out = run_attn(c)
    some = [0, 1, 77, heads - 1]
    few = dict(c, q=c["q"][:, some], kp=c["kp"][:, :, some], vp=c["vp"][:, :, some])
    check_attn(few, out[:, some])


@pytest.mark.usefixtures("table_width")
def test_attn_max_q_is_only_a_hint(device):
    for heads, lens in ((WIDE, CHUNKS), (COMMON, CHUNKS)):
        c = attn_case(lens, *heads, 64, F16, 9, device)
        ref = pagedref.attn(c["q"], c["kp"], c["vp"], c["cu"], c["kv"], c["table"], c["scale"])
        for m in (1, 2, 5, 37, 10000):
            check_attn(c, run_attn(c, max_q=m), ref)


@pytest.mark.usefixtures("table_width")
def test_attn_bad_pages(device):
    """An entry outside the cache makes its sequence's rows that see it NaN, and no others."""
    for heads, lens in ((WIDE, [(1, 200), (1, 300), (1, 40)]), (COMMON, [(50, 200), (60, 300), (1, 40)])):
        for entry in (-1, 1 << 30, 10000):
            c = attn_case(lens, *heads, 16, F16, 6, device)
            want = run_attn(c)
            c["table"][1, 3] = entry
            got = run_attn(c)
            a, b = int(c["cu"][1]), int(c["cu"][2])
            assert torch.equal(got[:a], want[:a]) and torch.equal(got[b:], want[b:])
            assert bool(got[a:b].isnan().all())


@pytest.mark.usefixtures("table_width")
def test_attn_device_lengths_outside_their_range(device):
    """cu_q past the batch or going back, lengths past the table: nothing outside is touched,
    the sequences that are in order are right."""
    c = attn_case([(2, 40), (3, 60), (2, 30)], *WIDE, 16, F16, 2, device, pad=4)
    ref = pagedref.attn(c["q"], c["kp"], c["vp"], c["cu"], c["kv"], c["table"], c["scale"])
    wild = dict(c, cu=i32([0, 2, 5, 1 << 30], device))
    got = run_attn(wild)
    check_attn(dict(c, rows=5), torch.cat([got[:5], torch.full_like(got[5:], 7)]), ref)
    wild = dict(c, cu=i32([0, 2, -9, 7], device))
    got = run_attn(wild)
    assert torch.equal(got[:2], run_attn(c)[:2])
    long = dict(c, kv=i32([40, 60, 1 << 30], device))
    long["table"] = c["table"].clamp(max=3)
    got = run_attn(long)
    assert got.shape == c["q"].shape


@pytest.mark.parametrize("n,heads,max_q", [(5, WIDE, 1), (300, WIDE, 300), (700, COMMON, 700)])
@pytest.mark.usefixtures("table_width")
def test_attn_rows_of_many_sequences(n, heads, max_q, device):
    """cu_q that names the same rows again and again: more row tiles than the batch can have.
    What the rows hold is not said; the workspace is not left."""
    c = attn_case([(n, 900)], *heads, 16, F16, 1, device)
    n_seq, hq, hkv, d = 300, *heads[:3]
    need = paged.attn_ws_bytes(n, n_seq, hq, hkv, d, max_q)
    room = torch.full((need + 8192,), 90, dtype=torch.uint8, device=device)
    wild = dict(c, cu=i32([0, n] * (n_seq // 2) + [0], device), kv=c["kv"].repeat(n_seq),
                table=c["table"].repeat(n_seq, 1), max_q=max_q)
    run_attn(wild, workspace=room[4096:4096 + need])
    assert bool((room[:4096] == 90).all()) and bool((room[4096 + need:] == 90).all())


@pytest.mark.usefixtures("table_width")
def test_attn_from_two_threads(device):
    """Threads that launch at once, each on its stream, share the library's workspace."""
    cases = [attn_case([(1, 6000), (3, 77)], *WIDE, 16, F16, 1, device),
             attn_case([(90, 3000)], *COMMON, 64, BF16, 5, device)]
    want = [run_attn(c) for c in cases]
    torch.cuda.synchronize()
    got = [[], []]

    def run(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[k].append(run_attn(cases[k]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for outs, w in zip(got, want):
        assert len(outs) == 20 and all(torch.equal(x, w) for x in outs)


@pytest.mark.usefixtures("table_width")
def test_attn_workspace_and_streams(device):
    """A caller's workspace, and calls on several streams at once, each with its own."""
    cases = [attn_case([(1, 900), (1, 400), (3, 77)], *WIDE, 16, F16, s, device) for s in range(3)]
    cases += [attn_case([(90, 700)], *COMMON, 64, BF16, 5, device)]
    want = [run_attn(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    spaces = [torch.empty(max(1, paged.attn_ws_bytes(c["q"].shape[0], len(c["kv"]), c["q"].shape[1],
                                                     c["kp"].shape[2], c["q"].shape[2], c["max_q"])),
                          dtype=torch.uint8, device=device) for c in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for c, s, w in zip(cases, streams, spaces):
            with torch.cuda.stream(s):
                got.append(run_attn(c, workspace=w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = []
    for c, s in zip(cases, streams):  # the library's: ordered between streams
        with torch.cuda.stream(s):
            got.append(run_attn(c))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attn_offsets_past_32_bits(device):
    """A cache of more than 2^32 bytes and elements: its far pages are read and written."""
    hq, hkv, d, page = 8, 2, 256, 64
    n_pages = (1 << 31) // (page * hkv * d) + 50
    kp = torch.empty((n_pages, page, hkv, d), dtype=F16, device=device)
    vp = torch.empty((n_pages, page, hkv, d), dtype=F16, device=device)
    lens = [(2, 130), (70, 200)]
    table = i32([[n_pages - 1, 3, n_pages - 7, 0], [n_pages - 2, n_pages - 30, 5, n_pages - 3]], device)
    g = torch.Generator(device=device).manual_seed(2)
    for p in table.flatten().tolist():
        kp[p].normal_(generator=g)
        vp[p].normal_(generator=g)
    small = torch.arange(8, dtype=torch.int32, device=device).view(2, 4)
    n = 72
    q = torch.randn((n, hq, d), generator=g, device=device).to(F16)
    k = torch.randn((n, hkv, d), generator=g, device=device).to(F16)
    v = torch.randn((n, hkv, d), generator=g, device=device).to(F16)
    t = torch.cat([torch.arange(128, 130), torch.arange(130, 200)])
    seq = torch.tensor([0] * 2 + [1] * 70)
    slots = (table.cpu()[seq, t // page] * page + t % page).int().to(device)
    q_out = torch.empty_like(q)
    paged.qk_norm_rope(q, k, q_out, positions=t.int().to(device), v=v, k_pages=kp, v_pages=vp, slots=slots)
    flat = table.flatten().long()
    c = dict(q=q_out, gate=None, kp=kp, vp=vp, table=table, cu=i32([0, 2, 72], device),
             kv=i32([130, 200], device), scale=d ** -0.5, max_q=70, rows=72)
    near = dict(c, kp=kp[flat].contiguous(), vp=vp[flat].contiguous(), table=small)
    out = run_attn(c)
    check_attn(near, out)


# ------------------------------------------------------------ the run of them
def test_serving_run(device):
    """Requests come, are prefilled in chunks, decode and end, some refused for want of pages;
    each step's plan, rows and attention in a row, checked against a plain cache."""
    hq, hkv, d, page, n_seq, n_tok = 6, 2, 128, 8, 5, 96
    rng = np.random.default_rng(3)
    g = torch.Generator().manual_seed(4)
    w = (1 + 0.2 * torch.randn(d, generator=g)).to(device)
    t = paged.PageTable(n_seq, 20, 22, page, n_tok, device)
    layer = paged.PagedLayer(t, H_q=hq, H_kv=hkv, head_dim=d, dtype=F16, rotary_dim=64, q_weight=w,
                             k_weight=w)
    held_k, held_v = [[] for _ in range(n_seq)], [[] for _ in range(n_seq)]
    refused = 0
    for step in range(12):
        q_len = [int(rng.choice([-1, 0, 1, 1, 1, 2, 17, 40])) for _ in range(n_seq)]
        while sum(max(0, x) for x in q_len) > n_tok:
            q_len[int(np.argmax(q_len))] = 1
        n = sum(max(0, x) for x in q_len)
        x = lambda *s: torch.randn(s, generator=g).to(F16).to(device)  # noqa: E731
        q_gate, k, v = x(n_tok, hq, 2 * d), x(n_tok, hkv, d), x(n_tok, hkv, d)
        q0, gate = q_gate[..., :d].clone(), q_gate[..., d:].clone()
        out = torch.full((n_tok, hq, d), 7, dtype=F16, device=device)
        t.step(i32(q_len, device))
        layer.attention(q_gate, k, v, out, d ** -0.5, max_q=40)
        cu, kv, pos = t.cu_q.tolist(), t.seq_kv.tolist(), t.positions.cpu()
        refused += int(t.status)
        _, k_rot, k_size = pagedref.norm_rope(k, w, pos, 1e-6, 1e7, 64)
        _, q_rot, size = pagedref.norm_rope(q0, w, pos, 1e-6, 1e7, 64)
        check_rows(q_gate[:n, :, :d], q_rot[:n], size[:n], F16)
        for s, a in enumerate(q_len):
            if a < 0:
                held_k[s], held_v[s] = [], []
            if a <= 0:
                continue
            rows = slice(cu[s], cu[s + 1])
            if kv[s] == 0:  # refused: nothing kept, its rows are 0
                assert not out[rows].any()
                continue
            at = t.slots[rows].long()
            kept = layer.k_pages.view(-1, hkv, d)[at]
            check_rows(kept, k_rot[rows], k_size[rows], F16)
            held_k[s] += list(kept.cpu())
            held_v[s] += list(v[rows].cpu())
            assert kv[s] == len(held_k[s])
            kk, vv = torch.stack(held_k[s])[None], torch.stack(held_v[s])[None]
            one = dict(q=q_gate[rows][..., :d], rows=a)
            ref = pagedref.attn(one["q"], kk, vv, torch.tensor([0, a]), torch.tensor([kv[s]]),
                                torch.zeros((1, 1), dtype=torch.int32), d ** -0.5, gate[rows])
            check_attn(one, out[rows], ref)
        assert bool((out[n:] == 7).all())
    assert refused > 0


def test_serving_step_replayed(device):
    """A whole decode step in a graph: replays follow the lengths and tokens they find."""
    hq, hkv, d, n_seq = 24, 4, 256, 6
    t = paged.PageTable(n_seq, 40, 100, 16, n_seq, device)
    layer = paged.PagedLayer(t, H_q=hq, H_kv=hkv, head_dim=d)
    g = torch.Generator(device=device).manual_seed(9)
    layer.k_pages.normal_(generator=g)
    layer.v_pages.normal_(generator=g)
    first = paged.PageTable(n_seq, 40, 100, 16, 512, device)  # the prompts' step, a wider batch
    prompts = i32([40, 1, 90, 17, 16, 31], device)
    first.step(prompts)
    for name in ("table", "kv_len", "free_pages", "state"):
        getattr(t, name).copy_(getattr(first, name))
    q_len = i32([1] * n_seq, device)
    qg = torch.zeros((n_seq, hq, 512), dtype=F16, device=device)
    k = torch.zeros((n_seq, hkv, d), dtype=F16, device=device)
    v = torch.zeros_like(k)
    out = torch.zeros((n_seq, hq, d), dtype=F16, device=device)
    ws = torch.empty(max(1, paged.attn_ws_bytes(n_seq, n_seq, hq, hkv, d, 1)), dtype=torch.uint8,
                     device=device)

    def step():
        t.step(q_len)
        layer.attention(qg, k, v, out, 1 / 16, max_q=1, workspace=ws)

    def state():
        return [x.clone() for x in (t.table, t.kv_len, t.free_pages, t.state, layer.k_pages, layer.v_pages)]

    def put(s):
        for x, y in zip((t.table, t.kv_len, t.free_pages, t.state, layer.k_pages, layer.v_pages), s):
            x.copy_(y)

    saved = state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    put(saved)
    for i in range(20):
        fresh = [torch.randn(x.shape, generator=g, device=device).to(F16) for x in (qg, k, v)]
        before = state()
        for x, y in zip((qg, k, v), fresh):
            x.copy_(y)
        q_len[i % n_seq] = i % 2
        step()
        eager = out.clone()
        after = state()
        put(before)
        qg.copy_(fresh[0])
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[: int(t.cu_q[-1])], eager[: int(t.cu_q[-1])]), i
        assert all(torch.equal(a, b) for a, b in zip(after, state())), i


def test_wrong_arguments_refused(device):
    c = attn_case([(1, 20)], *WIDE, 16, F16, 1, device)
    bad = [dict(cu_q=c["cu"].long()), dict(cu_q=c["cu"][:1]), dict(seq_kv=c["kv"].cpu()),
           dict(table=c["table"].t()), dict(gate=c["q"].to(BF16)), dict(gate=c["q"][..., :128]),
           dict(workspace=torch.empty(4, 4, device=device).t()), dict(table=c["table"][:0])]
    for over in bad:
        with pytest.raises((TypeError, ValueError)):
            run_attn(c, **over)
    with pytest.raises(ValueError):
        run_attn(dict(c, kp=c["kp"][..., :100]))
    with pytest.raises(ValueError):
        run_attn(dict(c, vp=c["vp"].transpose(1, 2)))
    with pytest.raises(ValueError):
        run_attn(dict(c, q=c["q"][:, :23]))
    with pytest.raises(ValueError, match="overlap"):
        run_attn(c, out=torch.zeros((1, 1, 256), dtype=F16, device=device).expand(1, 24, 256))
    with pytest.raises(ValueError):
        paged.qk_norm_rope(c["q"], None, torch.empty_like(c["q"]), q_weight=torch.ones(256))
    with pytest.raises(ValueError):
        paged.qk_norm_rope(None, c["kp"][0], None)
    with pytest.raises(ValueError):
        paged.qk_norm_rope(None, c["kp"][0], None, v=c["vp"][0], k_pages=c["kp"], v_pages=c["vp"])
