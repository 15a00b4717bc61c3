"""What a beam search refuses before anything runs, and statuses of its entry points that need no GPU."""
import ctypes
import math

import pytest
import torch

FAKE = ctypes.c_void_p(4096)


@pytest.fixture(scope="module")
def nat():
    from neuratensor_b200 import build, native
    build.build()
    native.load()
    return native


def select(L, dtype=1, B=2, K=3, V=100, n=3, x=FAKE, scores=FAKE, lengths=None, alpha=0.0, pad=0, stay=0, out=FAKE, ws=FAKE, nbytes=1 << 30):
    return L.nt_beam_select(dtype, B, K, V, n, x, V, scores, None, lengths, alpha, pad, stay, out, FAKE, FAKE, ws, nbytes, None)


@pytest.mark.parametrize("bad,status,text", [
    (dict(dtype=2), 2, "dtype"), (dict(K=0), 1, "beams"), (dict(K=65), 1, "beams"), (dict(n=0), 1, "wanted"), (dict(n=65), 1, "wanted"),
    (dict(V=0), 1, "sizes"), (dict(B=-1), 1, "sizes"), (dict(B=30000), 1, "65535"), (dict(n=2, stay=1), 1, "n == K"),
    (dict(alpha=math.nan), 1, "finite"), (dict(alpha=1.0), 1, "lengths"), (dict(pad=-1), 1, "pad"), (dict(x=None), 1, "null"),
    (dict(scores=None), 1, "null"), (dict(out=None), 1, "null"), (dict(ws=None), 6, "workspace"), (dict(nbytes=8), 6, "workspace"),
    (dict(x=ctypes.c_void_p(4097)), 1, "alignment")])
def test_select_status(nat, bad, status, text):
    L = nat.load()
    assert select(L, **bad) == status
    assert text in L.nt_last_error().decode()


def reorder(L, spec=((4096, 64, 64),), R=4, group=2, rows=FAKE):
    words = (ctypes.c_int64 * (3 * len(spec)))(*[v for s in spec for v in s])
    return L.nt_reorder_rows(len(spec), words, R, group, rows, None)


@pytest.mark.parametrize("bad,text", [
    (dict(group=0), "sizes"), (dict(group=3), "sizes"), (dict(R=2048, group=2048), "sizes"), (dict(R=-2), "sizes"), (dict(rows=None), "null"),
    (dict(spec=((0, 64, 64),)), "null"), (dict(spec=((4096, 64, 32),)), "rows of 64 bytes"), (dict(spec=((4096, -1, 32),)), "rows of -1")])
def test_reorder_status(nat, bad, text):
    L = nat.load()
    assert reorder(L, **bad) == 1
    assert text in L.nt_last_error().decode()


def fork(L, R=4, n=8, blocks=3, page=16, tokens=1, window=-1, group=2, table=FAKE, sb=3, shared=FAKE, ws=FAKE, nbytes=1 << 20):
    return L.nt_kv_fork(R, n, blocks, page, tokens, window, group, table, sb, FAKE, FAKE, FAKE, FAKE, shared, ws, nbytes, None)


@pytest.mark.parametrize("bad,status,text", [
    (dict(R=1025), 1, "at most 1024"), (dict(R=-1), 1, "rows"), (dict(page=0), 1, "sizes"), (dict(tokens=-1), 1, "sizes"),
    (dict(group=3), 1, "sizes"), (dict(sb=2), 1, "sizes"), (dict(blocks=1 << 28), 1, "sizes"), (dict(table=None), 1, "null"),
    (dict(shared=None), 1, "null"), (dict(ws=None), 6, "workspace"), (dict(nbytes=1), 6, "workspace")])
def test_fork_status(nat, bad, status, text):
    L = nat.load()
    assert fork(L, **bad) == status
    assert text in L.nt_last_error().decode()


def copy(L, spec=((4096,) * 4,), n=8, H=2, page=16, D=64, count=1, pages=FAKE):
    words = (ctypes.c_int64 * (4 * len(spec)))(*[v for s in spec for v in s])
    return L.nt_kv_copy_pages(len(spec), words, n, H, page, D, count, pages, None)


@pytest.mark.parametrize("bad,text", [
    (dict(H=0), "sizes"), (dict(n=-1), "sizes"), (dict(D=0), "sizes"), (dict(pages=None), "null"), (dict(spec=((4096, 0, 4096, 4096),)), "null"),
    (dict(spec=((4104, 4096, 4096, 4096),)), "alignment")])
def test_copy_status(nat, bad, text):
    L = nat.load()
    assert copy(L, **bad) == 1
    assert text in L.nt_last_error().decode()


def shared(L, dtype=1, B=4, groups=2, T=1, Hq=2, H=2, D=64, page=16, blocks=1 << 16, window=-1, q=FAKE, codes=FAKE, sh=FAKE, ws=None, nbytes=0):
    return L.nt_kv_attention_shared(dtype, B, groups, T, Hq, H, D, page, 4, blocks, window, 1.0, q, 0, 0, 0, codes, FAKE, FAKE, FAKE, FAKE,
                                    blocks, FAKE, None, sh, FAKE, ws, nbytes, None)


@pytest.mark.parametrize("bad,status,text", [
    (dict(groups=3), 1, "in 3 groups"), (dict(groups=0), 1, "groups"), (dict(dtype=7), 2, "dtype"), (dict(D=256), 1, "head_dim"),
    (dict(page=128), 1, "page"), (dict(Hq=3), 1, "sizes"), (dict(blocks=1 << 28), 1, "sizes"), (dict(q=None), 1, "null"), (dict(sh=None), 1, "null"),
    (dict(codes=ctypes.c_void_p(4104)), 1, "alignment"), (dict(), 6, "workspace")])
def test_shared_attention_status(nat, bad, status, text):
    L = nat.load()
    assert shared(L, **bad) == status
    assert text in L.nt_last_error().decode()


def test_workspaces_and_empty_calls(nat):
    L = nat.load()
    need = L.nt_kv_attention_shared_workspace_bytes(1, 4, 2, 1, 2, 2, 64, 16, 1 << 16, -1)
    assert need > 0 and shared(L, ws=FAKE, nbytes=need - 1) == 6
    # short reaches are the attention without sharing, which needs no more than that
    assert L.nt_kv_attention_shared_workspace_bytes(1, 4, 2, 1, 2, 2, 64, 16, 8, -1) == L.nt_kv_attention_workspace_bytes(4, 1, 2, 2, 64, 16, 8, -1)
    assert L.nt_kv_attention_shared_workspace_bytes(1, 4, 4, 1, 2, 2, 64, 16, 1 << 16, -1) == L.nt_kv_attention_workspace_bytes(4, 1, 2, 2, 64, 16, 1 << 16, -1)
    assert L.nt_kv_attention_shared_workspace_bytes(1, 4, 3, 1, 2, 2, 64, 16, 8, -1) == 0
    assert shared(L, B=0, q=None) == 0 and shared(L, T=0, q=None) == 0
    assert select(L, B=0, x=None) == 0 and reorder(L, R=0, rows=None) == 0 and reorder(L, spec=(), rows=None) == 0
    assert fork(L, R=0, table=None) == 0 and copy(L, count=0, pages=None) == 0 and copy(L, spec=(), pages=None) == 0
    assert L.nt_beam_select_workspace_bytes(1, 2, 3, 100, 3) > 0 and L.nt_beam_select_workspace_bytes(1, 2, 65, 100, 3) == 0
    assert L.nt_kv_fork_workspace_bytes(4, 3, 2) > 0 and L.nt_kv_fork_workspace_bytes(4, 3, 0) == 0


def test_packed_calls_of_a_beam_search(nat):
    """nt_call_packed reads the arguments in their order: the same refusals, by the argument that is wrong."""
    L = nat.load()

    def call(name, *args):
        entry, n, pack = nat._PACKED[name]
        words = pack(*args)
        assert len(words) == 8 * n
        return L.nt_call_packed(entry, words, n), L.nt_last_error().decode()

    X = 4096
    need = L.nt_beam_select_workspace_bytes(1, 2, 3, 100, 3)
    assert call("nt_beam_select", 1, 2, 3, 100, 3, X, 100, X, 0, 0, 0.0, 7, 1, X, X, X, X, need - 1, 0) == (
        6, f"nt_beam_select: workspace {need - 1} < {need} bytes")
    assert call("nt_beam_select", 1, 2, 3, 100, 3, X, 100, X, 0, 0, 0.5, 7, 1, X, X, X, X, need, 0)[1].endswith("needs lengths")
    assert call("nt_beam_select", 1, 2, 3, 100, 3, X, 100, X, 0, 0, 0.0, -7, 1, X, X, X, X, need, 0)[1].endswith("pad -7")
    assert call("nt_reorder_rows", 1, X, 4, 3, X, 0)[1].startswith("nt_reorder_rows: bad sizes")
    assert call("nt_reorder_rows", 0, 0, 4, 2, 0, 0)[0] == 0
    need = L.nt_kv_fork_workspace_bytes(4, 3, 2)
    assert call("nt_kv_fork", 4, 8, 3, 16, 1, -1, 2, X, 3, X, X, X, X, X, X, need - 1, 0) == (6, f"nt_kv_fork: workspace {need - 1} < {need} bytes")
    assert call("nt_kv_fork", 4, 8, 3, 16, 1, -1, 2, X, 3, X, X, 0, X, X, X, need, 0)[1].endswith("null pointer")
    assert call("nt_kv_copy_pages", 0, 0, 8, 2, 16, 64, 1, X, 0)[0] == 0
    assert call("nt_kv_copy_pages", 1, X, 8, 2, 16, 0, 1, X, 0)[1].endswith("bad sizes")
    need = L.nt_kv_attention_shared_workspace_bytes(1, 4, 2, 1, 2, 2, 64, 16, 1 << 16, -1)
    args = (1, 4, 2, 1, 2, 2, 64, 16, 4, 1 << 16, -1, 1.0, X, 0, 0, 0, X, X, X, X, X, 1 << 16, X, 0, X, X, X)
    assert call("nt_kv_attention_shared", *args, need - 1, 0) == (6, f"nt_kv_attention_shared: workspace {need - 1} < {need} bytes")


@pytest.mark.parametrize("more,text", [
    (dict(temperature=0.7), "temperature"), (dict(top_p=0.9), "top_p"), (dict(repetition_penalty=1.1), "repetition_penalty"),
    (dict(frequency_penalty=0.1), "frequency_penalty"), (dict(logit_bias={1: 1.0}), "logit_bias"),
    (dict(allowed=torch.ones(1, 70, dtype=torch.bool)), "allowed"), (dict(num_beams=0), "num_beams"), (dict(num_beams=65), "num_beams"),
    (dict(num_beams=-3), "num_beams"), (dict(length_penalty=math.inf), "length_penalty"), (dict(stop_tokens=[70]), "stop_tokens"),
    (dict(max_new_tokens=0), "new token"), (dict(num_beams=1, length_penalty=1.0), "num_beams above 1")])
def test_generate_refuses_what_a_beam_search_does_not_take(more, text):
    from neuratensor_b200 import ModelConfig, NeuraTensorModel
    model = NeuraTensorModel(ModelConfig(vocab_size=70, d_model=128, n_layers=2, d_state=16, max_seq_len=64, attn_every=2,
                                         attn_heads=2, attn_window=8))
    with pytest.raises(ValueError, match=text):
        model.generate(torch.zeros(2, 3, dtype=torch.int64), **{**dict(max_new_tokens=2, num_beams=2), **more})
    with pytest.raises(ValueError, match="1024"):
        model.generate(torch.zeros(600, 3, dtype=torch.int64), max_new_tokens=2, num_beams=2)
