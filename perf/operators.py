"""The paged-cache operators: what their speed is measured on.

A server that decodes many conversations at once keeps the keys and values of
its uncompressed layers in pages of a fixed number of tokens.  Each step of
such a server takes three operators:

  plan   from the number of new tokens of each request: its new pages off the
         free list, its block table, and for each new token its position and
         the cache slot it goes to;
  rows   the new tokens' query and key heads normalised and rotated to their
         positions, keys and values written to their slots;
  attn   the new tokens' attention over the pages, each token seeing its
         request's tokens up to itself, the output gated.

`step` is the three in a row.  Head counts and widths are the engine's 24 / 4
x 256 with 64 rotated dims, and a common 32 / 8 x 128 with every dim rotated.

With `own` false the operators are computed in their plain form: elementary
torch operations in 32 bits (angles in 64), rounded once at the end.
`exact` is written from the definitions in 64 bits, one request at a time.
"""
import math
import os
import random
import sys

import torch

own = False  # set by whoever measures: false the plain forms, true the framework's operators

DEV = "cuda"
THETA = 1e7
EPS = 1e-6
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
# head layouts: query heads, KV heads, width, rotated dims, a gate beside each query
HEADS = {"wide": (24, 4, 256, 64, True), "common": (32, 8, 128, 128, False)}

MAX_SEQS, MAX_ROWS, MAX_CTX, MAX_PROMPT, MAX_POS = 512, 65536, 131072, 8192, 262144


def _paged():
    """The framework's operators (imported only where they are measured)."""
    package = os.path.abspath("bonsai-mojo-1bit-optimization-t4-cuda_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from khq import paged

    return paged


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # A decode step of a loaded server: 64 requests, a token each, a few of
        # them at a page's end.  The smallest call, where its latency counts.
        {"name": "plan_64", "kind": "plan", "n_seq": 64, "q_lo": 1, "q_hi": 1, "ctx_lo": 100,
         "ctx_hi": 8192, "ended": 0, "page": 16, "mix": 1},
        # The same server's busiest step: 512 requests, decoding, prefilling,
        # idle and ended ones among them, some 50,000 new tokens.
        {"name": "plan_512", "kind": "plan", "n_seq": 512, "q_lo": 1, "q_hi": 700, "ctx_lo": 1,
         "ctx_hi": 16384, "ended": 9, "page": 64, "mix": 2},
        # The rows of a decode step of 32 conversations.
        {"name": "rows_32", "kind": "rows", "heads": "wide", "dtype": "fp16", "n": 32, "page": 64,
         "pos": 20000},
        # A prompt of 8,192 tokens, the largest chunk a prefill pass takes.
        {"name": "rows_8192", "kind": "rows", "heads": "wide", "dtype": "fp16", "n": MAX_PROMPT,
         "page": 64, "pos": MAX_POS},
        # An odd number of rows in bfloat16, every dim rotated, far positions.
        {"name": "rows_bf16_1999", "kind": "rows", "heads": "common", "dtype": "bf16", "n": 1999,
         "page": 48, "pos": MAX_POS},
        # One conversation's decode step at 512 tokens: launches and latency.
        {"name": "attn_512", "kind": "attn", "heads": "wide", "dtype": "fp16", "n_seq": 1, "q_lo": 1,
         "q_hi": 1, "ctx_lo": 511, "ctx_hi": 511, "page": 16, "mix": 3},
        # 32 ragged conversations of 1K to 16K tokens decoded together.
        {"name": "attn_batch_32", "kind": "attn", "heads": "wide", "dtype": "fp16", "n_seq": 32,
         "q_lo": 1, "q_hi": 1, "ctx_lo": 1024, "ctx_hi": 16384, "page": 64, "mix": 5},
        # One decode step at the longest context, an odd length.
        {"name": "attn_131071", "kind": "attn", "heads": "wide", "dtype": "fp16", "n_seq": 1,
         "q_lo": 1, "q_hi": 1, "ctx_lo": MAX_CTX - 2, "ctx_hi": MAX_CTX - 2, "page": 128, "mix": 6},
        # A chunk of 128 tokens after 8,192: chunked prefill.
        {"name": "attn_chunk_128", "kind": "attn", "heads": "wide", "dtype": "fp16", "n_seq": 1,
         "q_lo": 128, "q_hi": 128, "ctx_lo": 8192, "ctx_hi": 8192, "page": 64, "mix": 7},
        # A whole prompt of 8,192 tokens in one call.  The largest case.
        {"name": "attn_prompt_8192", "kind": "attn", "heads": "wide", "dtype": "fp16", "n_seq": 1,
         "q_lo": MAX_PROMPT, "q_hi": MAX_PROMPT, "ctx_lo": 0, "ctx_hi": 0, "page": 64, "mix": 8},
        # Continuous batching in bfloat16: chunks and decoding requests in one
        # call, pages of 48 tokens that end inside the kernels' tiles.
        {"name": "attn_mixed_bf16", "kind": "attn", "heads": "common", "dtype": "bf16", "n_seq": 24,
         "q_lo": 1, "q_hi": 700, "ctx_lo": 1, "ctx_hi": 9000, "page": 48, "mix": 9},
        # A whole decode step of 16 conversations: plan, rows and attention.
        {"name": "step_16", "kind": "step", "heads": "wide", "dtype": "fp16", "n_seq": 16, "q_lo": 1,
         "q_hi": 1, "ctx_lo": 300, "ctx_hi": 6000, "page": 64, "mix": 10},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = {"kind": rng.choice(["plan", "rows", "attn", "attn", "attn", "step"]),
             "page": rng.choice([16, 16, 32, 48, 64, 64, 100, 128]), "mix": rng.randrange(1 << 20)}
        if c["kind"] != "plan":
            c["heads"] = rng.choice(["wide", "wide", "common"])
            c["dtype"] = rng.choice(["fp16", "bf16"])
        if c["kind"] == "rows":
            c["n"] = _log(rng, 1, MAX_PROMPT)
            c["pos"] = _log(rng, 1000, MAX_POS)
        elif c["kind"] == "plan":
            c["n_seq"] = _log(rng, 1, MAX_SEQS)
            c["q_lo"], c["q_hi"] = 1, _log(rng, 1, 700)
            c["ctx_lo"], c["ctx_hi"] = 1, _log(rng, 64, 16384)
            c["ended"] = rng.randrange(0, 10)
            if sum(max(0, n) for n in _lengths(c)[0]) > MAX_ROWS:
                continue
        elif c["kind"] == "step" or rng.random() < 0.5:  # decode, or a few tokens each
            c["n_seq"] = _log(rng, 1, 64)
            c["q_lo"], c["q_hi"] = 1, rng.choice([1, 1, 1, 2, 5])
            c["ctx_hi"] = _log(rng, 64, max(64, min(MAX_CTX, 600000 // c["n_seq"])))
            c["ctx_lo"] = max(1, c["ctx_hi"] // rng.choice([1, 3, 16]))
        else:  # prefill and continuous batching
            c["n_seq"] = _log(rng, 1, 24)
            c["q_hi"] = _log(rng, 16, MAX_PROMPT // c["n_seq"])
            c["q_lo"] = max(1, c["q_hi"] // rng.choice([1, 4, 1000]))
            c["ctx_lo"] = 0
            c["ctx_hi"] = _log(rng, 1, 16384)
        if _cost(c) <= most and _padded(c) <= 2.0e9:
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _padded(case):
    """Values of the plain form's padded scores."""
    if case["kind"] not in ("attn", "step"):
        return 0
    q, ctx = _lengths(case)
    return len(q) * max(q) * HEADS[case["heads"]][0] * max(a + b for a, b in zip(q, ctx))


def _lengths(case):
    """New tokens (-1: the request has ended) and tokens held of each request."""
    rng = random.Random(case["mix"])
    q, ctx = [], []
    for _ in range(case["n_seq"]):
        n = _log(rng, case["q_lo"], case["q_hi"])
        if rng.randrange(100) < case.get("ended", 0):
            n = rng.choice([-1, 0])
        q.append(n)
        ctx.append(0 if case["ctx_hi"] == 0 else _log(rng, max(1, case["ctx_lo"]), case["ctx_hi"]))
    return q, ctx


def work(case):
    if case["kind"] == "rows":
        return _rows_work(case, case["n"])
    q, ctx = _lengths(case)
    new = [max(0, n) for n in q]
    if case["kind"] == "plan":
        return _plan_work(case, q, ctx)
    hq, hkv, d, _, gated = HEADS[case["heads"]]
    n = sum(new)
    pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(new, ctx))
    held = sum(a + b for a, b in zip(new, ctx) if a)
    total = {"bytes": 2 * n * hq * d * (3 if gated else 2) + 4 * held * hkv * d,
             "flops": 4 * d * hq * pairs}
    if case["kind"] == "step":
        for w in (_plan_work(case, q, ctx), _rows_work(case, n)):
            total = {k: total[k] + w[k] for k in total}
    return total


def _plan_work(case, q, ctx):
    page = case["page"]
    pages = sum(-(-(a + b) // page) - -(-b // page) if a > 0 else (-(-b // page) if a < 0 else 0)
                for a, b in zip(q, ctx))
    n = sum(max(0, a) for a in q)
    return {"bytes": 8 * n + 4 * 5 * len(q) + 8 * pages + 16, "flops": 4 * n + 8 * len(q)}


def _rows_work(case, n):
    hq, hkv, d, rot, _ = HEADS[case["heads"]]
    return {"bytes": 2 * 2 * n * (hq + 2 * hkv) * d + 8 * n + 8 * d,
            "flops": n * (hq + hkv) * (4 * d + 3 * rot)}


# ------------------------------------------------------------------ the inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _empty(*shape):
    return torch.zeros(shape, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": dict(case)}
    if case["kind"] == "rows":
        n, page = case["n"], case["page"]
        _tokens(s, case, n, g)
        n_pages = -(-n // page) + 1
        _pages(s, case, n_pages, g)
        # a run of tokens: its pages in no order, its first slot inside a page
        order = torch.randperm(n_pages, generator=g, device=DEV)
        at = torch.arange(n, device=DEV) + page // 3
        s["slots"] = (order[at // page] * page + at % page).to(torch.int32)
        s["positions"] = torch.randint(0, case["pos"], (n,), generator=g, device=DEV,
                                       dtype=torch.int32)
        return s
    q, ctx = _lengths(case)
    page, n_seq = case["page"], case["n_seq"]
    step = case["kind"] == "step"
    width = max(-(-(max(0, a) + b) // page) for a, b in zip(q, ctx)) + 2
    n_pages = sum(-(-(max(0, a) + b) // page) for a, b in zip(q, ctx)) + 5
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    held = [-(-b // page) if case["kind"] != "attn" else -(-(a + b) // page) for a, b in zip(q, ctx)]
    # the requests' pages, then the free ones
    cu = torch.tensor([0] + held, device=DEV).cumsum(0)
    cols = torch.arange(width, device=DEV)
    index = (cu[:-1, None] + cols).clamp(max=n_pages - 1)
    s["table"] = torch.where(cols < _i32(held)[:, None], order[index], 0).to(torch.int32)
    n_tok = sum(max(0, a) for a in q)
    if case["kind"] == "plan":
        n_tok += 37  # a padded batch
    if case["kind"] != "attn":
        taken = sum(held)
        # the free list is a ring: its first entry somewhere in it
        head = n_pages // 3
        at = (torch.arange(n_pages - taken, device=DEV) + head) % n_pages
        s["free"] = _empty(n_pages)
        s["free"][at] = order[taken:]
        s["state"] = _i32([head, n_pages - taken])
        s["q_len"], s["kv_len"] = _i32(q), _i32(ctx)
        s.update(cu_q=_empty(n_seq + 1), seq_kv=_empty(n_seq), kv_out=_empty(n_seq),
                 state_out=_empty(2), status=_empty(1), positions=_empty(n_tok), slots=_empty(n_tok))
    else:
        s["cu_q"] = _i32([0] + q).cumsum(0).to(torch.int32)
        s["seq_kv"] = _i32([a + b for a, b in zip(q, ctx)])
    if case["kind"] == "plan":
        return s
    s["max_q"] = max(q)
    _pages(s, case, n_pages, g)
    _tokens(s, case, n_tok, g)
    if not step:  # normalised and rotated already: peaked as a trained model's queries are
        s["q"].mul_(1.5)
    s["out"] = torch.zeros_like(s["q_out"])
    return s


def _tokens(s, case, n, g):
    """The projections of n tokens: queries, their gates beside them, keys and values."""
    hq, hkv, d, _, gated = HEADS[case["heads"]]
    dt = DTYPES[case["dtype"]]
    if gated:
        q_gate = torch.randn((n, hq, 2 * d), generator=g, device=DEV, dtype=dt)
        s["q"], s["gate"] = q_gate[..., :d], q_gate[..., d:]
    else:
        s["q"], s["gate"] = torch.randn((n, hq, d), generator=g, device=DEV, dtype=dt), None
    s["q_out"] = torch.zeros((n, hq, d), device=DEV, dtype=dt)
    if case["kind"] != "attn":
        s["k"] = torch.randn((n, hkv, d), generator=g, device=DEV, dtype=dt) * 3
        s["v"] = torch.randn((n, hkv, d), generator=g, device=DEV, dtype=dt)
        s["q_w"] = 1 + 0.2 * torch.randn(d, generator=g, device=DEV)
        s["k_w"] = 1 + 0.2 * torch.randn(d, generator=g, device=DEV)


def _pages(s, case, n_pages, g):
    _, hkv, d, _, _ = HEADS[case["heads"]]
    shape = (n_pages, case["page"], hkv, d)
    dt = DTYPES[case["dtype"]]
    s["k_pages"] = torch.randn(shape, generator=g, device=DEV, dtype=dt)
    s["v_pages"] = torch.randn(shape, generator=g, device=DEV, dtype=dt)


# ------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    steps = {"plan": [_plan], "rows": [_rows], "attn": [_attn], "step": [_plan, _rows, _attn]}[kind]
    out = {}
    for op in steps:
        out.update(op(state))
    return out


def _plan(s):
    page, n_tok = s["case"]["page"], s["slots"].shape[0]
    if own:
        _paged().plan(s["q_len"], s["kv_len"], s["table"], s["free"], s["state"], page_size=page,
                      cu_q=s["cu_q"], seq_kv=s["seq_kv"], kv_out=s["kv_out"],
                      state_out=s["state_out"], status=s["status"], positions=s["positions"],
                      slots=s["slots"])
        names = ("table", "free", "cu_q", "seq_kv", "kv_out", "state_out", "status", "positions",
                 "slots")
        return {k: s[k] for k in names}
    q, kv, table, free = s["q_len"].long(), s["kv_len"].long(), s["table"], s["free"]
    n_pages, width = free.shape[0], table.shape[1]
    new = q.clamp(min=0)
    ends = new.cumsum(0)
    has, want = (kv + page - 1) // page, (kv + new + page - 1) // page
    fits = (want <= width) & (ends <= n_tok) & (new > 0)
    need = torch.where(fits, want - has, 0)
    upto = need.cumsum(0)
    head, count = s["state"][0].long(), s["state"][1].long()
    taken_ok = fits & ((need == 0) | (upto <= count))
    taken = torch.where(taken_ok, upto, 0).amax()
    # new pages into the block table
    cols = torch.arange(width, device=DEV)
    fresh = (cols >= has[:, None]) & (cols < want[:, None]) & taken_ok[:, None]
    ring = (head + (upto - need)[:, None] + cols - has[:, None]) % n_pages
    table = torch.where(fresh, free[ring], table)
    # pages of ended requests onto the free list
    back = torch.where(q < 0, has, 0)
    first = back.cumsum(0) - back
    i = torch.arange(n_pages, device=DEV)
    off = (i - head - count) % n_pages
    seq = torch.searchsorted(first + back, off, right=True).clamp(max=len(q) - 1)
    from_seq = table[seq, (off - first[seq]).clamp(0, width - 1)]
    free = torch.where(off < back.sum(), from_seq, free)
    # each token's request, position and slot
    cu = torch.cat([ends.new_zeros(1), ends]).clamp(max=n_tok)
    t = torch.arange(n_tok, device=DEV)
    seq = torch.searchsorted(cu[1:], t, right=True)
    real = seq < len(q)
    seq = seq.clamp(max=len(q) - 1)
    pos = torch.where(real, kv[seq] + t - cu[seq], 0)
    at = table[seq, (pos // page).clamp(max=width - 1)].long()
    slots = torch.where(real & taken_ok[seq], at * page + pos % page, -1)
    made = {"table": table, "free": free, "cu_q": cu.int(),
            "seq_kv": torch.where(taken_ok, kv + new, torch.where(q == 0, kv, 0)).int(),
            "kv_out": torch.where(taken_ok, kv + new, torch.where(q < 0, 0, kv)).int(),
            "state_out": torch.stack([(head + taken) % n_pages, count - taken + back.sum()]).int(),
            "status": ((new > 0) & ~taken_ok).sum().int().reshape(1),
            "positions": pos.int(), "slots": slots.int()}
    s["made"] = made  # what the next operators of a step read
    return made


def _rows(s):
    c = s["case"]
    _, _, d, rot, _ = HEADS[c["heads"]]
    if own:
        _paged().qk_norm_rope(s["q"], s["k"], s["q_out"], positions=s["positions"], q_weight=s["q_w"],
                              k_weight=s["k_w"], eps=EPS, theta=THETA, rotary_dim=rot, v=s["v"],
                              k_pages=s["k_pages"], v_pages=s["v_pages"], slots=s["slots"])
        return {k: s[k] for k in ("q_out", "k_pages", "v_pages")}
    made = s.get("made", s)
    half = rot // 2
    freq = torch.exp(-math.log(THETA) / half * torch.arange(half, device=DEV, dtype=torch.float64))
    angle = made["positions"].double()[:, None, None] * freq
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def turned(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b = x[..., :half], x[..., half:rot]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., rot:]], -1)

    s["q_out"].copy_(turned(s["q"], s["q_w"]))
    slots = made["slots"].long()
    for pages, new in (("k_pages", turned(s["k"], s["k_w"]).to(s["k"].dtype)), ("v_pages", s["v"])):
        s[pages].view(-1, *new.shape[1:])[slots] = new
    return {k: s[k] for k in ("q_out", "k_pages", "v_pages")}


def _attn(s):
    c = s["case"]
    hq, hkv, d, _, _ = HEADS[c["heads"]]
    q = s["q_out"] if c["kind"] == "step" else s["q"]
    if own:
        _paged().attn(q, s["k_pages"], s["v_pages"], s["out"], cu_q=s["cu_q"], seq_kv=s["seq_kv"],
                      table=s["table"], max_q=s["max_q"], scale=d ** -0.5, gate=s["gate"])
        return {"out": s["out"]}
    made = s.get("made", s)
    page, table, rep = c["page"], made["table"].long(), hq // hkv
    n_seq, max_q = table.shape[0], s["max_q"]
    cu, kv = made["cu_q"].long(), made["seq_kv"].long()
    longest = max(a + b for a, b in zip(*_lengths(c)))  # what a server knows of its batch
    n, keys = q.shape[0], torch.arange(longest, device=DEV)
    at = table[:, keys // page] * page + keys % page
    # padded to one batch: keys of each request, and its queries by KV head
    k = s["k_pages"].view(-1, hkv, d)[at].permute(0, 2, 1, 3).float()
    v = s["v_pages"].view(-1, hkv, d)[at].permute(0, 2, 1, 3).float()
    new = cu[1:] - cu[:-1]
    i = torch.arange(max_q, device=DEV)
    rows = (cu[:-1, None] + i).clamp(max=n - 1)
    x = q[rows].float().view(n_seq, max_q, hkv, rep, d).permute(0, 2, 3, 1, 4)
    x = x.reshape(n_seq, hkv, rep * max_q, d)
    sees = (kv - new)[:, None] + i + 1  # keys a query sees
    mask = keys < sees[:, :, None]
    p = torch.matmul(x, k.transpose(2, 3).contiguous()).mul_(d ** -0.5)
    p = p.view(n_seq, hkv, rep, max_q, longest).masked_fill_(~mask[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    # a request's keys past its end are another's or none: no weight, and no value either
    v = v.masked_fill((keys >= kv[:, None])[:, None, :, None], 0)
    o = torch.matmul(p.view(n_seq, hkv, rep * max_q, longest), v).view(n_seq, hkv, rep, max_q, d)
    o = torch.where(total > 0, o / total, 0).permute(0, 3, 1, 2, 4).reshape(n_seq, max_q, hq, d)
    t = torch.arange(n, device=DEV)
    seq = torch.searchsorted(cu[1:], t, right=True).clamp(max=n_seq - 1)
    o = o[seq, t - cu[seq]]
    if s["gate"] is not None:
        o = o / (1 + torch.exp(-s["gate"].float()))
    return {"out": o.to(q.dtype)}


# ----------------------------------------------------------------- in 64 bits
def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    hq, hkv, d, rot, _ = HEADS[case["heads"]]
    if case["kind"] == "attn":
        return {"out": _exact_attn(s, s["q"], s["k_pages"], s["v_pages"], s["table"])}
    page = case["page"]
    if case["kind"] == "step":  # tokens go to the requests' next slots, pages as the ring has them
        q_len, ctx = _lengths(case)
        free, state, table = s["free"].tolist(), s["state"].tolist(), s["table"].tolist()
        at, slots, positions = state[0], [], []
        for row, a, b in zip(table, q_len, ctx):
            for pos in range(b, b + a):
                if pos % page == 0:
                    row[pos // page] = free[at % len(free)]
                    at += 1
                slots.append(row[pos // page] * page + pos % page)
                positions.append(pos)
        table = _i32(table)
        s["slots"], s["positions"] = _i32(slots), _i32(positions)
    pairs = torch.arange(rot // 2, device=DEV, dtype=torch.float64)
    angle = s["positions"].double().unsqueeze(1) * THETA ** (-2 * pairs / rot)
    turn = torch.polar(torch.ones_like(angle), angle).unsqueeze(1)

    def rows(x, w):
        x = x.double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / d + EPS).sqrt() * w.double()
        z = torch.complex(x[..., : rot // 2], x[..., rot // 2: rot]) * turn
        return torch.cat([z.real, z.imag, x[..., rot:]], -1)

    q, k = rows(s["q"], s["q_w"]), rows(s["k"], s["k_w"])
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    page_of, in_page = s["slots"].long() // page, s["slots"].long() % page
    k_pages[page_of, in_page] = k
    v_pages[page_of, in_page] = s["v"].double()
    out = {"q_out": q, "k_pages": k_pages, "v_pages": v_pages}
    if case["kind"] == "step":
        # the attention reads what the cache and the query buffer hold: values of the type
        dt = DTYPES[case["dtype"]]
        out["out"] = _exact_attn(s, q.to(dt), k_pages.to(dt), v_pages.to(dt), table)
    return out


def _exact_attn(s, q, k_pages, v_pages, table):
    case = s["case"]
    hq, hkv, d, _, _ = HEADS[case["heads"]]
    out, at = torch.zeros(q.shape, dtype=torch.float64, device=DEV), 0
    for row, a, b in zip(table, *_lengths(case)):
        if a <= 0:
            continue
        pages = row[: -(-(a + b) // case["page"])].long()
        k = k_pages[pages].reshape(-1, hkv, d)[: a + b].double()
        v = v_pages[pages].reshape(-1, hkv, d)[: a + b].double()
        unseen = torch.ones((a, a + b), dtype=torch.bool, device=DEV).triu_(b + 1)
        for h in range(hq):
            g = h * hkv // hq
            score = q[at: at + a, h].double() @ k[:, g].t().contiguous() / math.sqrt(d)
            weight = torch.softmax(score.masked_fill_(unseen, -math.inf), 1)
            out[at: at + a, h] = weight @ v[:, g].contiguous()
        at += a
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())
