"""The generation-step operators among differentiated ones (B200)."""
import pytest
import torch

from test_gpu_step_ops import BF16, DEV, F32, U32, close, freqs, gen, make_cache, nat, rotary64  # noqa: F401

pytestmark = pytest.mark.gpu


def calls(nat, x):  # noqa: F811
    """One call of each operator that writes what it is given, on x [2, 3, 4, 64] or as many numbers of it."""
    rows = x.view(2, -1)
    tokens = torch.zeros(2, 3, device=DEV, dtype=torch.int64)
    return {"rotary": lambda: nat.rotary(x, torch.arange(3, device=DEV), freqs(64), out=x),
            "rotary into": lambda: nat.rotary(torch.ones_like(x), torch.arange(3, device=DEV), freqs(64), out=x),
            "logits": lambda: nat.logits_process(rows, tokens=tokens, repetition=2.0, out=rows),
            "logits into": lambda: nat.logits_process(torch.ones_like(rows), tokens=tokens, repetition=2.0, out=rows)}


@pytest.mark.parametrize("which", ["rotary", "rotary into", "logits", "logits into"])
def test_a_saved_tensor_that_is_written_is_known(nat, which):  # noqa: F811
    """torch's own in-place operations raise in a backward pass that saved what they wrote; so do these."""
    w = torch.randn(2, 3, 4, 64, device=DEV, generator=gen(60), requires_grad=True)
    x = w * 2
    loss = (x * x).sum()                                     # saves x
    with torch.no_grad():
        calls(nat, x)[which]()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_a_saved_cache_that_is_written_is_known(nat):  # noqa: F811
    cache, table = make_cache(1, 2, 3, 16, 64, 61)
    w = torch.ones(4, 3, device=DEV, requires_grad=True)
    n = torch.ones(1, device=DEV, dtype=torch.int32)
    k = torch.randn(1, 1, 3, 64, device=DEV, generator=gen(62))
    for i in (1, 3):
        loss = (w * cache[i]).sum()
        versions = [t._version for t in cache]
        nat.kv_append(k, k, *cache, table, n)
        assert all(t._version > v for t, v in zip(cache, versions))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    versions = [t._version for t in cache]
    nat.kv_attention(k, *cache, table, n)
    assert [t._version for t in cache] == versions


@pytest.mark.parametrize("which", ["rotary into", "logits into"])
def test_writing_a_tensor_that_requires_grad_is_refused(nat, which):  # noqa: F811
    x = torch.randn(2, 3, 4, 64, device=DEV, generator=gen(63), requires_grad=True)
    before = x.detach().clone()
    with pytest.raises(RuntimeError, match="requires grad"):
        calls(nat, x)[which]()
    assert torch.equal(x, before)
    with torch.no_grad():
        calls(nat, x)[which]()                               # as torch's own allow it
    assert not torch.equal(x, before)


def test_a_cache_that_requires_grad_is_refused(nat):  # noqa: F811
    cache, table = make_cache(1, 2, 3, 16, 64, 64)
    k, n = torch.ones(1, 1, 3, 64, device=DEV), torch.ones(1, device=DEV, dtype=torch.int32)
    cache[1].requires_grad_()
    with pytest.raises(RuntimeError, match="requires grad"):
        nat.kv_append(k, k, *cache, table, n)


def test_inference_tensors_are_written(nat):  # noqa: F811
    """They have no version; writing them is as before, captured too."""
    with torch.inference_mode():
        x = torch.ones(2, 3, 4, 64, device=DEV)
        for call in calls(nat, x).values():
            call()
        cache, table = make_cache(1, 2, 3, 16, 64, 65)
        k, n = torch.ones(1, 1, 3, 64, device=DEV), torch.ones(1, device=DEV, dtype=torch.int32)
        nat.kv_append(k, k, *cache, table, n)
        assert cache[0][table[0, 0].long(), :, 0].float().eq(256).all()          # 1 / 2^-8


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_derivatives(nat, dtype, layout):  # noqa: F811
    """The map is linear: the tangent is the rotation of the tangent."""
    import torch.autograd.forward_ad as fwd
    x = torch.randn(2, 3, 4, 64, device=DEV, generator=gen(66)).to(dtype)
    t = torch.randn(2, 3, 4, 64, device=DEV, generator=gen(67)).to(dtype)
    pos, f = torch.randint(0, 5000, (2, 3), device=DEV, generator=gen(68)), freqs(48)
    turn = lambda x: nat.rotary(x, pos, f, layout=layout, mscale=0.9)  # noqa: E731
    y, want = turn(x), turn(t)
    with fwd.dual_level():
        for off in (False, True):                            # forward mode goes on under no_grad
            with torch.set_grad_enabled(off):
                got = fwd.unpack_dual(turn(fwd.make_dual(x, t)))
            assert torch.equal(got.primal, y) and torch.equal(got.tangent, want)
    back = nat.rotary(t, pos, f, layout=layout, mscale=0.9, inverse=True)
    with pytest.raises(RuntimeError):                        # not taken by torch.func, and said so
        torch.func.jvp(turn, (x,), (t,))
    with pytest.raises(RuntimeError):
        torch.func.vjp(turn, x)
    # backwards, and a second time: the gradient is linear in dy
    leaf, dy = x.clone().requires_grad_(), t.clone().requires_grad_()
    (g,) = torch.autograd.grad(turn(leaf), leaf, dy, create_graph=True)
    assert torch.equal(g, back)
    (gg,) = torch.autograd.grad(g, dy, x)
    assert torch.equal(gg, y)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_gradient_in_bf16(nat, layout):  # noqa: F811
    B, T, H, D, R, m = 2, 9, 3, 64, 40, 0.9
    g = gen(69)
    x = torch.randn(B, T, H, D, device=DEV, generator=g).to(BF16).requires_grad_()
    dy = torch.randn(B, T, H, D, device=DEV, generator=g).to(BF16)
    pos, f = torch.randint(0, 5000, (B, T), device=DEV, generator=g), freqs(R)
    (gx,) = torch.autograd.grad(nat.rotary(x, pos, f, layout=layout, mscale=m), x, dy)
    want, mag = rotary64(dy, pos, f, layout, m, inverse=True)
    close(gx, want, torch.finfo(BF16).eps / 2, 8 * U32 * mag)


def test_derivatives_that_do_not_exist_are_refused(nat):  # noqa: F811
    """Backwards and forwards, by every floating argument, and nothing is written."""
    import torch.autograd.forward_ad as fwd
    cache, table = make_cache(1, 2, 3, 16, 64, 74)
    k, n = torch.ones(1, 1, 3, 64, device=DEV), torch.ones(1, device=DEV, dtype=torch.int32)
    rows, tokens = torch.randn(2, 40, device=DEV, generator=gen(75)), torch.zeros(2, 3, device=DEV, dtype=torch.int64)
    per_row, ids = torch.ones(2, device=DEV), torch.zeros(2, 1, device=DEV, dtype=torch.int64)
    pos, f = torch.arange(1, device=DEV), freqs(64)
    names = ("k_codes", "k_scale", "v_codes", "v_scale")
    pool = dict(zip(names, cache), table=table, lengths=n)
    cases = [(nat.kv_append, dict(k=k, v=k, **pool), ("k", "v", "k_scale", "v_scale")),
             (nat.kv_attention, dict(q=k, **pool), ("q", "k_scale", "v_scale")),
             (nat.logits_process, dict(logits=rows, tokens=tokens, repetition=per_row, frequency=per_row, presence=per_row,
                                       bias_ids=ids, bias=per_row[:, None]),
              ("logits", "repetition", "frequency", "presence", "bias")),
             (nat.logits_process, dict(logits=rows, out=torch.empty_like(rows)), ("logits", "out")),
             (nat.rotary, dict(x=k, positions=pos, inv_freq=f, out=torch.empty_like(k)), ("x", "inv_freq", "out")),
             (nat.rotary, dict(x=k, positions=pos, inv_freq=f), ("inv_freq",))]
    before = [t.clone() for t in cache]
    for fn, good, floating in cases:
        for name in floating:
            with pytest.raises(RuntimeError, match="backward|gradient|requires grad"):
                fn(**{**good, name: good[name].clone().requires_grad_()})
            with fwd.dual_level(), pytest.raises(RuntimeError, match="forward|backward|gradient"):
                fn(**{**good, name: fwd.make_dual(good[name].clone(), torch.ones_like(good[name]))})
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, before))
    for fn, good, _ in cases:                                # and without any they run
        fn(**good)
        with fwd.dual_level():
            fn(**good)
