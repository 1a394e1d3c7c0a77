"""The embedding's, the losses' and AdamW's host side, without a GPU: argument statuses of every entry point, workspaces, the
differentiable functions' dealings with autograd (their operators replaced by plain torch), the optimizer's arguments."""

import ctypes

import pytest
import torch

F32, I64, BF16, I32 = 0, 1, 2, 3


@pytest.fixture(scope="module")
def lib():
    from omarchy_mac_torch import _lib
    return _lib


def test_embedding_statuses(lib):
    L, p, bad, no, ok = lib.L, ctypes.c_void_p(4096), lib.OMT_INVALID, lib.OMT_UNSUPPORTED, lib.OMT_OK
    f = L.omt_embedding_fwd
    assert f(I64, I64, 4, 8, 16, p, p, 1.0, p, None) == bad
    assert f(F32, F32, 4, 8, 16, p, p, 1.0, p, None) == bad  # tokens that are no integers
    assert f(F32, I64, -1, 8, 16, p, p, 1.0, p, None) == bad
    assert f(F32, I64, 4, 0, 16, p, p, 1.0, p, None) == bad
    assert f(F32, I64, 4, 8, 0, p, p, 1.0, p, None) == bad
    assert f(F32, I32, 4, 8, 16, None, p, 1.0, p, None) == bad
    assert f(F32, I32, 0, 8, 16, None, None, 1.0, None, None) == ok
    b, ws = L.omt_embedding_bwd, L.omt_embedding_bwd_workspace
    assert b(F32, I64, 4000, 8, 16, p, p, -1, 1.0, p, None, 0, None) == bad  # no workspace
    assert b(F32, I64, 4000, 8, 16, p, p, -1, 1.0, p, p, ws(4000, 8, 16) - 1, None) == bad
    assert b(F32, I64, 4000, 8, 16, p, p, -1, 1.0, p, ctypes.c_void_p(4100), 1 << 30, None) == bad
    assert b(F32, I64, 4, 8, 16, p, p, -1, 1.0, None, p, 1 << 30, None) == bad
    assert b(F32, I64, 4, 8, 16, None, p, -1, 1.0, p, p, 1 << 30, None) == bad
    assert b(F32, I64, (1 << 28) + 1, 8, 16, p, p, -1, 1.0, p, p, 1 << 40, None) == no
    assert b(F32, I64, 4, 8, (1 << 16) + 1, p, p, -1, 1.0, p, p, 1 << 40, None) == no
    assert b(F32, I64, 4, (1 << 28) + 1, 16, p, p, -1, 1.0, p, p, 1 << 40, None) == no
    # sorted tokens and positions twice, each run's two sums
    assert ws(100000, 50000, 1024) >= 4 * 4 * 100000 and ws(-1, 8, 16) == 0
    assert ws(100, 8, 16) == ws(2048, 256, 128) == 0 < ws(2049, 256, 128)  # few positions are sorted in LDS


def logits(lib, sequences=2, length=3, vocab=10, dtype=F32, x=4096, labels=4096):
    return ctypes.byref(lib.Logits(x, labels, -100, sequences, length, vocab, length * vocab, vocab, dtype))


def test_loss_statuses(lib):
    L, p, bad, no, ok = lib.L, ctypes.c_void_p(4096), lib.OMT_INVALID, lib.OMT_UNSUPPORTED, lib.OMT_OK
    f, b = L.omt_token_logps_fwd, L.omt_token_logps_bwd
    assert f(None, p, p, None) == bad
    for wrong in (dict(dtype=I64), dict(sequences=-1), dict(vocab=0), dict(x=None), dict(labels=None)):
        assert f(logits(lib, **wrong), p, p, None) == bad and b(logits(lib, **wrong), p, p, p, None) == bad
    assert f(logits(lib, length=1 << 28), p, p, None) == no
    assert f(logits(lib, vocab=(1 << 28) + 1), p, p, None) == no
    assert f(logits(lib), None, p, None) == bad and f(logits(lib), p, None, None) == bad
    assert b(logits(lib), p, None, p, None) == bad and b(logits(lib), p, p, None, None) == bad
    for empty in (dict(sequences=0, x=None, labels=None), dict(length=0, x=None, labels=None)):
        assert f(logits(lib, **empty), None, None, None) == ok and b(logits(lib, **empty), None, None, None, None) == ok

    need = L.omt_preference_workspace(2, 3)
    g = lambda q, ref=p, kind=0, beta=0.1, smooth=0.0, loss=p, rewards=p, ws=p, size=need: \
        L.omt_preference_loss(q, ref, kind, beta, smooth, 0, loss, rewards, p, ws, size, None)  # noqa: E731
    assert g(logits(lib, sequences=3)) == bad and g(logits(lib, sequences=0)) == bad
    assert g(logits(lib), kind=3) == bad and g(logits(lib), kind=-1) == bad
    assert g(logits(lib), beta=0.0) == bad and g(logits(lib), beta=float("nan")) == bad
    assert g(logits(lib), kind=1, smooth=0.1) == bad and g(logits(lib), kind=2, smooth=0.1) == bad
    assert g(logits(lib), smooth=-0.1) == bad and g(logits(lib), smooth=1.1) == bad
    assert g(logits(lib), ref=None) == bad and g(logits(lib), loss=None) == bad and g(logits(lib), rewards=None) == bad
    assert g(logits(lib), ws=None) == bad and g(logits(lib), size=need - 1) == bad
    assert g(logits(lib), ws=ctypes.c_void_p(4104)) == bad
    assert g(logits(lib, sequences=1 << 23, length=1), size=1 << 40) == no
    assert L.omt_preference_workspace(1 << 20, 1 << 20) == 0

    need = L.omt_policy_workspace(2, 3, 1)
    h = lambda q, old=p, adv=p, lo=0.2, hi=0.2, loss=p, kl=p, logps=p, ws=p, size=need: \
        L.omt_policy_loss(q, old, None, adv, 1, 0, lo, hi, 0.0, 1, loss, kl, logps, p, ws, size, None)  # noqa: E731
    assert h(logits(lib), old=None) == bad and h(logits(lib), adv=None) == bad and h(logits(lib), logps=None) == bad
    assert h(logits(lib), loss=None) == bad and h(logits(lib), kl=None) == bad
    assert h(logits(lib), lo=-0.1) == bad and h(logits(lib), hi=float("nan")) == bad
    assert h(logits(lib), ws=None) == bad and h(logits(lib), size=need - 1) == bad
    assert h(logits(lib, length=1 << 28)) == no and h(logits(lib, sequences=1 << 22, length=1), size=1 << 40) == no
    assert L.omt_policy_workspace(-1, 3, 0) == 0

    s = L.omt_scale_by
    assert s(I64, 4, p, p, None) == bad and s(F32, -1, p, p, None) == bad and s(F32, 4, None, p, None) == bad
    assert s(BF16, 0, None, None, None) == ok


def test_adamw_statuses(lib):
    L, bad, no, ok = lib.L, lib.OMT_INVALID, lib.OMT_UNSUPPORTED, lib.OMT_OK
    hp = lib.AdamwParams(1e-3, 0.9, 0.999, 0.01, 1e-8, None, None, None, 0)

    def f(tensors, dtype=F32, bits=32, params=hp, count=None):
        arr = (lib.AdamwTensor * max(1, len(tensors)))(*tensors)
        return L.omt_adamw(dtype, bits, ctypes.byref(params) if params else None, arr, len(tensors) if count is None else count, None)

    def t(param=4096, grad=4096, master=None, m=4096, ms=4096, v=4096, vs=4096, step=4096, n=0):
        return lib.AdamwTensor(param, grad, master, m, ms, v, vs, step, n)

    assert f([]) == ok and f([t()]) == ok
    assert f([t()], dtype=I64) == bad and f([t()], bits=16) == bad and f([t()], params=None) == bad and f([], count=-1) == bad
    for missing in (dict(param=None), dict(grad=None), dict(m=None), dict(v=None), dict(step=None)):
        assert f([t(n=5, **missing)]) == bad
    for missing in (dict(ms=None), dict(vs=None)):
        assert f([t(n=5, **missing)], bits=8) == bad
    assert f([t(n=-1)]) == bad and f([t(n=1 << 40)]) == no
    assert f([t(master=4096, n=5)]) == bad                               # a master copy of float32
    assert f([t(master=4096, n=5), t(n=5)], dtype=BF16) == bad           # of some alone


def test_operators_refuse_cpu_tensors_and_wrong_choices():
    from omarchy_mac_torch import hip_ops as ops
    x, labels = torch.ones(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64)
    for call in (lambda: ops.embedding(labels, x[0]), lambda: ops.embedding_backward(x, labels, 4),
                 lambda: ops.token_logps(x, labels), lambda: ops.token_logps_backward(x[..., 0], x, labels, x[..., 0]),
                 lambda: ops.preference_loss(x, labels, x[:, 0, 0]), lambda: ops.policy_loss(x, labels, x[..., 0], x[:, 0, 0]),
                 lambda: ops.adamw([x], [x], [x], [x], x[0, 0, 0])):
        with pytest.raises(TypeError, match="HIP device"):
            call()
    with pytest.raises(ValueError, match="kind"):
        ops.preference_loss(x, labels, x[:, 0, 0], kind="other")
    with pytest.raises(ValueError, match="reduction"):
        ops.policy_loss(x, labels, x[..., 0], x[:, 0, 0], reduction="batch")
    for row in (4, -5):
        with pytest.raises(ValueError, match="padding_idx"):
            ops.embedding_backward(x, labels, 4, padding_idx=row)
    ops.adamw([], [], [], [], x[0, 0, 0])


@pytest.fixture
def plain_losses(monkeypatch):
    """hip_ops' losses in plain torch, with a record of whether a gradient was asked for."""
    from omarchy_mac_torch import hip_ops
    asked = []

    def preference(logits, labels, reference, grad=True, **_):
        asked.append(grad)
        return logits.sum(), reference * 2, torch.ones_like(logits) if grad else None

    def policy(logits, labels, old_logps, advantages, grad=True, **_):
        asked.append(grad)
        return logits.sum(), old_logps.sum(), old_logps * 1, torch.ones_like(logits) if grad else None

    monkeypatch.setattr(hip_ops, "preference_loss", preference)
    monkeypatch.setattr(hip_ops, "policy_loss", policy)
    monkeypatch.setattr(hip_ops, "scale_by_", lambda x, f: x.mul_(f))
    return asked


def test_losses_compute_a_gradient_only_where_one_can_be_asked_for(plain_losses):
    from omarchy_mac_torch import lm
    x, labels, ref = torch.ones(2, 3, 5, requires_grad=True), torch.zeros(2, 3, dtype=torch.int64), torch.ones(2)
    for call, others in ((lambda t: lm.preference_loss(t, labels, ref), 1),
                         (lambda t: lm.policy_loss(t, labels, torch.ones(2, 3), ref), 2)):
        plain_losses.clear()
        out = call(x)
        assert len(out) == 1 + others and out[0].requires_grad and not any(t.requires_grad for t in out[1:])
        with torch.no_grad():
            assert len(call(x)) == 1 + others
        call(x.detach())
        assert plain_losses == [True, False, False]
        (3 * out[0]).backward()
        assert torch.equal(x.grad, torch.full_like(x, 3.0))
        x.grad = None


def test_a_losss_gradient_is_handed_on_once(plain_losses):
    from omarchy_mac_torch import lm
    x, labels, ref = torch.ones(2, 3, 5, requires_grad=True), torch.zeros(2, 3, dtype=torch.int64), torch.ones(2)
    loss, _ = lm.preference_loss(x, labels, ref)
    loss.backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="runs once"):
        loss.backward()


def test_padding_rows_are_checked():
    from omarchy_mac_torch import lm
    with pytest.raises(ValueError, match="padding_idx"):
        lm.embedding(torch.zeros(2, dtype=torch.int64), torch.ones(4, 8), padding_idx=4)


def test_optimizer_arguments():
    from omarchy_mac_torch import optim
    p = [torch.nn.Parameter(torch.ones(3))]
    for wrong in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            optim.AdamW(p, **wrong)
    opt = optim.AdamW(p)
    opt.step()  # no gradients: nothing to do
    assert not opt.state
    p[0].grad = torch.ones(3)
    with pytest.raises(TypeError, match="HIP device"):
        opt.step()


def test_optimizer_states_are_float32_whatever_the_default(monkeypatch):
    from omarchy_mac_torch import hip_ops, optim
    monkeypatch.setattr(hip_ops, "adamw", lambda *args, **options: None)
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    opt = optim.AdamW([p])
    torch.set_default_dtype(torch.float64)
    try:
        opt.step()
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(opt.state[p][name].dtype == torch.float32 for name in ("step", "exp_avg_scale", "exp_avg_sq_scale"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 32])
def test_optimizer_states_keep_their_types_through_a_state_dict(monkeypatch, dtype, bits):
    from omarchy_mac_torch import hip_ops, optim
    monkeypatch.setattr(hip_ops, "adamw", lambda *args, **options: None)
    def made():
        p = torch.nn.Parameter(torch.linspace(-1, 1, 130).to(dtype))
        p.grad = torch.ones_like(p)
        return p, optim.AdamW([p], state_bits=bits)

    p, opt = made()
    opt.step()
    state = opt.state[p]
    held = torch.float8_e4m3fn if bits == 8 else torch.float32
    assert state["exp_avg"].dtype == state["exp_avg_sq"].dtype == held and state["exp_avg"].shape == p.shape
    assert ("exp_avg_scale" in state) == (bits == 8) and ("master" in state) == (dtype == torch.bfloat16)
    if bits == 8:
        assert state["exp_avg_scale"].shape == state["exp_avg_sq_scale"].shape == (2,)
    if "master" in state:
        state["master"] += 1e-5  # what the parameter's type cannot hold
    q, other = made()
    other.load_state_dict(opt.state_dict())
    assert other.state[q].keys() == state.keys() and float(other.state[q]["step"]) == 1
    for name, t in state.items():
        mine = other.state[q][name]
        assert mine.dtype == t.dtype and torch.equal(mine.float(), t.float()) and mine.data_ptr() != t.data_ptr()


def test_statuses_of_log_probabilities_in_64_bits(lib):
    L, p, bad, no, ok = lib.L, ctypes.c_void_p(4096), lib.OMT_INVALID, lib.OMT_UNSUPPORTED, lib.OMT_OK
    f, b = L.omt_token_logps_fwd64, L.omt_token_logps_bwd64
    assert f(None, p, p, None) == bad and b(None, p, p, p, None) == bad
    for wrong in (dict(dtype=I64), dict(sequences=-1), dict(vocab=0), dict(x=None), dict(labels=None)):
        assert f(logits(lib, **wrong), p, p, None) == bad and b(logits(lib, **wrong), p, p, p, None) == bad
    assert f(logits(lib, length=1 << 28), p, p, None) == no and b(logits(lib, vocab=(1 << 28) + 1), p, p, p, None) == no
    assert f(logits(lib), None, p, None) == bad and f(logits(lib), p, None, None) == bad
    assert b(logits(lib), None, p, p, None) == bad and b(logits(lib), p, None, p, None) == bad and b(logits(lib), p, p, None, None) == bad
    assert f(logits(lib, length=0, x=None), None, None, None) == ok and b(logits(lib, length=0, x=None), None, None, None, None) == ok


def test_embedding_takes_what_torchs_does():
    """from_pretrained, types, devices and options; on the host torch's results times the scale."""
    from omarchy_mac_torch import lm
    w, t = torch.randn(5, 4), torch.tensor([[0, 3], [4, 4]])
    for args, options in (((w,), {}), ((w, False), {}), ((w,), dict(freeze=False, padding_idx=3)), ((w, True, 1), dict(max_norm=0.5)),
                          ((w, False), dict(sparse=True)), ((w, False), dict(scale_grad_by_freq=True))):
        m, plain = lm.Embedding.from_pretrained(*args, scale=2.0, **options), torch.nn.Embedding.from_pretrained(*args, **options)
        assert isinstance(m, lm.Embedding) and m.scale == 2.0 and m.weight.requires_grad == plain.weight.requires_grad
        assert m.padding_idx == plain.padding_idx and torch.equal(m(t), 2 * plain(t))
        if m.weight.requires_grad:
            m(t).sum().backward()
            (2 * plain(t)).sum().backward()
            assert m.weight.grad.is_sparse == plain.weight.grad.is_sparse
            assert torch.equal(m.weight.grad.to_dense(), plain.weight.grad.to_dense())
    assert lm.Embedding.from_pretrained(w).scale == 1.0
    m = lm.Embedding(5, 4, dtype=torch.float64, device="cpu", scale=3.0)
    assert m.weight.dtype == torch.float64 and torch.equal(m(t), 3 * m.weight[t])
    assert lm.Embedding(5, 4, 2, 0.5).scale == 0.5 and lm.Embedding(5, 4, -1).padding_idx == 4
    with pytest.raises(TypeError):
        lm.Embedding(5, 4, other=1)


@pytest.fixture
def plain_embedding(monkeypatch):
    """hip_ops' embedding and its gradient in plain torch, without autograd, as the operators are."""
    from omarchy_mac_torch import hip_ops

    def embedding(tokens, weight, scale=1.0):
        with torch.no_grad():
            known = (tokens >= 0) & (tokens < len(weight))
            return torch.where(known[..., None], weight[tokens.clamp(0, len(weight) - 1)] * scale, float("nan"))

    def embedding_backward(gy, tokens, vocab, scale=1.0, padding_idx=None):
        with torch.no_grad():
            on = (tokens >= 0) & (tokens < vocab) & (tokens != (-1 if padding_idx is None else padding_idx % vocab))
            return torch.zeros(vocab, gy.shape[-1], dtype=gy.dtype).index_add_(0, tokens[on], gy[on]) * scale

    monkeypatch.setattr(hip_ops, "embedding", embedding)
    monkeypatch.setattr(hip_ops, "embedding_backward", embedding_backward)


@pytest.mark.parametrize("padding_idx", [None, 2, -1])
def test_embeddings_derivatives_of_any_order(plain_embedding, padding_idx):
    from torch.autograd import forward_ad
    from torch.autograd.gradcheck import gradcheck, gradgradcheck
    from omarchy_mac_torch import lm
    g = torch.Generator().manual_seed(0)
    w = torch.randn(5, 3, generator=g, dtype=torch.float64, requires_grad=True)
    v = torch.randn(5, 3, generator=g, dtype=torch.float64)
    t = torch.tensor([[0, 2, 2], [4, 1, 0]])
    mine = lambda w: lm.embedding(t, w, 1.5, padding_idx)  # noqa: E731
    plain = lambda w: 1.5 * torch.nn.functional.embedding(t, w, padding_idx)  # noqa: E731
    if padding_idx is None:  # (the padding row has a value but by definition no gradient)
        assert gradcheck(mine, w, check_forward_ad=True) and gradgradcheck(mine, w, check_fwd_over_rev=True)
    for f in (lambda f: torch.autograd.functional.hvp(lambda w: f(w).pow(3).sum(), w, v)[1],
              lambda f: torch.func.grad(lambda w: f(w).pow(3).sum())(w),
              lambda f: torch.func.jvp(f, (w,), (v,))[1],
              lambda f: torch.func.vmap(lambda a: f(w * a))(torch.arange(3.0, dtype=torch.float64)),
              lambda f: torch.func.vmap(torch.func.grad(lambda w: f(w).pow(2).sum()))(torch.stack([w, v]))):
        assert torch.allclose(f(mine), f(plain), rtol=1e-12, atol=0)
    for f in (lm.embedding, lambda t, w, s, p: s * torch.nn.functional.embedding(t, w, p)):  # by samples of tokens
        rows = torch.func.vmap(lambda row: f(row, w, 1.5, padding_idx))(t)
        each = torch.func.vmap(torch.func.grad(lambda w, row: f(row, w, 1.5, padding_idx).pow(2).sum()), (None, 0))(w, t)
        assert torch.equal(rows, 1.5 * w[t])
        assert torch.allclose(each.sum(0), torch.func.grad(lambda w: plain(w).pow(2).sum())(w), rtol=1e-12, atol=0)
    assert torch.equal(*(torch.autograd.functional.jacobian(f, w.detach()) for f in (mine, plain)))
    vs = torch.randn(4, 2, 3, 3, generator=g, dtype=torch.float64)  # several of the result's gradients at once
    mine_, plain_ = (torch.func.vmap(lambda v, y=f(w): torch.autograd.grad(y, w, v, retain_graph=True)[0])(vs) for f in (mine, plain))
    assert torch.allclose(mine_, plain_, rtol=1e-12, atol=0)
    with forward_ad.dual_level():
        y = forward_ad.unpack_dual(mine(forward_ad.make_dual(w.detach(), v)))
        assert torch.equal(y.tangent, 1.5 * v[t])


def test_tokens_outside_the_vocabulary_have_no_second_derivative(plain_embedding):
    from omarchy_mac_torch import lm
    w, t = torch.ones(4, 2, requires_grad=True), torch.tensor([1, 7, -1])
    x = torch.ones(3, 2, requires_grad=True)
    gw, = torch.autograd.grad(lm.embedding(t, w), w, x, create_graph=True)
    gx, = torch.autograd.grad((gw * torch.tensor(3.0)).sum(), x)
    assert gx.tolist() == [[3, 3], [0, 0], [0, 0]]


def test_a_refused_step_is_not_counted():
    from omarchy_mac_torch import optim
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    opt = optim.AdamW([p])
    for _ in range(2):
        with pytest.raises(TypeError, match="HIP device"):
            opt.step()
        assert float(opt.state[p]["step"]) == 0


def test_optimizer_loads_what_its_hooks_give_it(monkeypatch):
    """A hook before may replace the state dictionary, one after may change the states that were loaded."""
    from omarchy_mac_torch import hip_ops, optim
    monkeypatch.setattr(hip_ops, "adamw", lambda *args, **options: None)
    p, q = (torch.nn.Parameter(torch.linspace(-1, 1, 130).bfloat16()) for _ in range(2))
    p.grad = torch.ones_like(p)
    opt, other = optim.AdamW([p]), optim.AdamW([q])
    opt.step()
    saved = opt.state_dict()

    def before(_, d):
        state = {k: v | {"master": v["master"] + 1e-5, "step": v["step"] + 4} for k, v in d["state"].items()}
        return {"state": state, "param_groups": d["param_groups"]}

    def after(o):
        o.state[q]["step"] *= 2

    other.register_load_state_dict_pre_hook(before)
    other.register_load_state_dict_post_hook(after)
    for _ in range(2):
        other.load_state_dict(saved)
        assert other.state[q]["master"].dtype == torch.float32 and float(other.state[q]["step"]) == 10
        assert torch.equal(other.state[q]["master"], opt.state[p]["master"] + 1e-5)
        assert other.state[q]["exp_avg"].dtype == torch.float8_e4m3fn
    assert float(opt.state[p]["step"]) == 1
    with pytest.raises(ValueError):
        other.load_state_dict({"state": {}, "param_groups": []})


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optimizer_goes_on_from_torchs_states(monkeypatch, dtype):
    """torch's states stay in 32 bits; a parameter that had none gets this optimizer's; each kind is a call of its own."""
    from omarchy_mac_torch import hip_ops, optim
    calls = []
    monkeypatch.setattr(hip_ops, "adamw", lambda *args, **options: calls.append((args, options)))
    ps = [torch.nn.Parameter(torch.ones(3, dtype=dtype)) for _ in range(2)]
    theirs = torch.optim.AdamW(ps, lr=0.5, betas=(0.5, 0.75), weight_decay=0.25, fused=False)
    ps[0].grad = torch.full_like(ps[0], 0.5)
    theirs.step()
    opt = optim.AdamW(ps, state_bits=8)
    opt.load_state_dict(theirs.state_dict())
    ps[1].grad = torch.ones_like(ps[1])
    opt.step()
    assert len(calls) == 2
    for (args, options), p, bits, step in zip(calls, ps, (32, 8), (2, 1)):
        params, _, m, v, steps, ms, vs, masters = args
        assert params[0] is p and float(steps[0]) == step and (options["lr"], options["betas"]) == (0.5, (0.5, 0.75))
        held = torch.float32 if bits == 32 else torch.float8_e4m3fn
        assert m[0].dtype == v[0].dtype == held and (ms is None) == (vs is None) == (bits == 32)
        assert (masters is not None) == (bits == 8 and dtype == torch.bfloat16)
    assert opt.state[ps[0]]["exp_avg"].tolist() == [0.25] * 3
    theirs = torch.optim.AdamW(ps, amsgrad=True, fused=False)
    with pytest.raises(ValueError, match="amsgrad"):
        opt.load_state_dict(theirs.state_dict())
    assert opt.param_groups[0]["lr"] == 0.5


def test_optimizer_arguments_of_groups():
    from omarchy_mac_torch import optim
    p, q = (torch.nn.Parameter(torch.ones(3)) for _ in range(2))
    opt = optim.AdamW([p])
    for wrong in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            optim.AdamW([dict(params=[p], **wrong)])
        with pytest.raises(ValueError):
            opt.add_param_group(dict(params=[q], **wrong))
        with pytest.raises(ValueError):
            optim.AdamW([dict(params=[p], lr=1e-2, betas=(0.5, 0.5), eps=0.0, weight_decay=0.0, state_bits=8)], **wrong)
        assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[q], state_bits=32, lr=0.5))
    assert opt.param_groups[1]["state_bits"] == 32 and opt.param_groups[1]["betas"] == opt.defaults["betas"]
