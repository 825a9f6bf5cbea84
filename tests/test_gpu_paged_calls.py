"""The paged calls behind the native checks: what they take gives the Python function's
results, and what they do not take its errors, word for word, before anything is launched."""
import pytest
import torch

from khq import paged
from khq._lib import KhqError

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
N, H_Q, H_KV, D, PAGE, N_PAGES, N_SEQ = 6, 4, 2, 64, 16, 8, 2


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def half(*shape, seed=0, dtype=torch.float16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(DEV, dtype)


def arguments(name):
    """Good arguments of a call, all by name; and the tensors that it writes."""
    pages = dict(k_pages=half(N_PAGES, PAGE, H_KV, D, seed=1), v_pages=half(N_PAGES, PAGE, H_KV, D, seed=2))
    z = dict(device=DEV, dtype=torch.int32)
    if name == "plan":
        a = dict(q_len=i32(5, 1), kv_len=i32(30, 0), table=torch.zeros((N_SEQ, 4), **z),
                 free_pages=torch.arange(N_PAGES, **z), state=i32(0, N_PAGES), page_size=PAGE,
                 cu_q=torch.zeros(3, **z), seq_kv=torch.zeros(2, **z), kv_out=torch.zeros(2, **z),
                 state_out=torch.zeros(2, **z), status=torch.zeros(1, **z),
                 positions=torch.zeros(N, **z), slots=torch.zeros(N, **z))
        return a, ["table", "free_pages", "cu_q", "seq_kv", "kv_out", "state_out", "status",
                   "positions", "slots"]
    if name == "qk_norm_rope":
        a = dict(q=half(N, H_Q, D, seed=3), k=half(N, H_KV, D, seed=4), q_out=half(N, H_Q, D),
                 positions=i32(*range(7, 7 + N)), q_weight=torch.ones(D, device=DEV),
                 k_weight=torch.ones(D, device=DEV), eps=1e-5, theta=1e4, rotary_dim=32,
                 k_out=half(N, H_KV, D), k_normed=half(N, H_KV, D), v=half(N, H_KV, D, seed=5),
                 slots=i32(*range(N)), **pages)
        return a, ["q_out", "k_out", "k_normed", "k_pages", "v_pages"]
    a = dict(q=half(N, H_Q, D, seed=6), out=half(N, H_Q, D), cu_q=i32(0, 5, 6), seq_kv=i32(35, 1),
             table=i32(1, 2, 3, 4, 5, 6, 7, 0).view(N_SEQ, 4), max_q=5, scale=0.125,
             gate=half(N, H_Q, D, seed=7), **pages)
    return a, ["out"]


def outcome(f, a):
    try:
        return f(**a)
    except Exception as e:  # noqa: BLE001  (both sides' are compared)
        return type(e), str(e)


def wrong(name):
    return {
        "plan": dict(q_len=[None, 3, torch.zeros(2), i32(1), i32(1, 2, 3), torch.zeros(2, dtype=torch.int32)],
                     kv_len=[None, torch.zeros(2, device=DEV), i32(1), i32(0, 0, 0, 0)[::2]],
                     table=[None, i32(0, 0), torch.zeros((3, 4), dtype=torch.int32, device=DEV),
                            torch.zeros((4, 2), dtype=torch.int32, device=DEV).t()],
                     free_pages=[None, torch.zeros(8, device=DEV)], state=[i32(0)], page_size=[0, -1, 1 << 31],
                     cu_q=[i32(0, 0)], seq_kv=[i32(0)], kv_out=[i32(0)], state_out=[i32(0, 0, 0)],
                     status=[None], positions=[None, torch.zeros(N, device=DEV)], slots=[i32(0)],
                     stream=[7], unknown=[1]),
        "qk_norm_rope": dict(
            q=[3, torch.zeros((N, H_Q, D)), torch.zeros((N, H_Q, D), device=DEV), half(N, H_Q, 96),
               half(N, H_Q * D), half(N, H_Q, D, dtype=torch.bfloat16)],
            k=[3, half(N + 1, H_KV, D), half(N, H_KV + 1, D), half(N, D, H_KV).transpose(1, 2)],
            q_out=[None, half(N, H_KV, D), half(N, 1, D).expand(N, H_Q, D), half(N, H_Q, 2 * D)[..., ::2]],
            positions=[i32(0), torch.zeros(N, device=DEV)], pos0=[-1],
            q_weight=[half(D), torch.ones(D), torch.ones(2 * D, device=DEV)[::2]],
            k_weight=[torch.ones(D + 1, device=DEV)], eps=[-1.0, float("nan")], theta=[0.0],
            rotary_dim=[8, 128, -16], k_out=[half(1, H_KV, D).expand(N, H_KV, D)], k_normed=[half(N, H_Q, D)],
            v=[None, half(N, H_Q, D)], k_pages=[None, half(N_PAGES, PAGE, H_Q, D), half(N_PAGES, PAGE, H_KV, 128)],
            v_pages=[None, half(N_PAGES, PAGE, H_KV, D, dtype=torch.bfloat16)], slots=[None, i32(0)],
            unknown=[1]),
        "attn": dict(
            q=[None, half(N, 3, D), half(N, H_Q, 128), half(N, H_Q, D, dtype=torch.bfloat16), torch.zeros((N, H_Q, D))],
            k_pages=[None, half(N_PAGES, PAGE, D), half(N_PAGES, PAGE, H_KV, D + 4)[..., :D], half(0, PAGE, H_KV, D)],
            v_pages=[None, half(N_PAGES, PAGE, H_KV, D)[:, ::2], half(N_PAGES, PAGE, D, H_KV).transpose(2, 3)],
            out=[None, half(N, H_KV, D), half(1, H_Q, D).expand(N, H_Q, D)], cu_q=[None, i32(0, 1)],
            seq_kv=[i32(0)], table=[None, i32(0, 1), torch.zeros((0, 4), dtype=torch.int32, device=DEV)],
            max_q=[0, -1], gate=[half(N, H_KV, D)],
            workspace=[torch.zeros(4, device=DEV), torch.zeros(1 << 20), torch.zeros((64, 64), device=DEV).t()],
            unknown=[1]),
    }[name]


@pytest.mark.parametrize("name", ["plan", "qk_norm_rope", "attn"])
def test_refused_alike(name):
    call = getattr(paged, name)
    for arg, values in wrong(name).items():
        for i, value in enumerate(values):
            print(name, arg, i, flush=True)
            a, _ = arguments(name)
            a[arg] = value
            got, want = outcome(call, a), outcome(call.__wrapped__, a)
            assert got == want and isinstance(got, tuple), (arg, i, got, want)


@pytest.mark.parametrize("name", ["plan", "qk_norm_rope", "attn"])
def test_left_out_arguments(name):
    call = getattr(paged, name)
    good, _ = arguments(name)
    for arg in good:
        a = {k: v for k, v in good.items() if k != arg}
        assert outcome(call, a) == outcome(call.__wrapped__, a), arg
    with pytest.raises(TypeError):
        call()
    with pytest.raises(TypeError):
        call(*good.values())


@pytest.mark.parametrize("name", ["plan", "qk_norm_rope", "attn"])
@pytest.mark.parametrize("form", ["names", "positions", "stream", "numbers", "status"])
def test_same_results(name, form):
    call = getattr(paged, name)
    left = []
    for f in (call, call.__wrapped__):
        a, outs = arguments(name)
        args = ()
        if form == "positions":
            n = {"plan": 5, "qk_norm_rope": 3, "attn": 0}[name]
            args = [a.pop(k) for k in list(a)[:n]]
        elif form == "stream":
            a["stream"] = torch.cuda.Stream()
            a["stream"].wait_stream(torch.cuda.current_stream())
        elif form == "numbers":
            a.update({"plan": {}, "qk_norm_rope": dict(eps=1, theta=10000), "attn": dict(scale=1)}[name])
        elif form == "status":
            a["check"] = False
        assert f(*args, **a) == 0
        torch.cuda.synchronize()
        a.update(zip(list(arguments(name)[0]), args))
        left.append([a[k] for k in outs])
    for x, y, k in zip(*left, outs):
        assert torch.equal(x, y), k


def test_status_of_a_refused_call():
    a, _ = arguments("attn")
    a.update(max_q=0, check=False)
    assert paged.attn(**a) == paged.attn.__wrapped__(**a) == -100
    a["check"] = True
    with pytest.raises(KhqError, match="khq_paged_attn"):
        paged.attn(**a)


def test_on_a_current_stream():
    a, _ = arguments("attn")
    paged.attn(**a)
    want = a["out"].clone()
    a["out"].zero_()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        paged.attn(**a)
        got = a["out"].clone()
    s.synchronize()
    assert torch.equal(got, want)
