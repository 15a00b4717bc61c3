"""Refusals of the generation-step entry points that need no GPU: a status and a message, never an abort."""
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


def rotary(L, dtype=0, B=1, T=2, H=3, D=64, R=64, x=FAKE, y=FAKE, pos=FAKE, freq=FAKE, ys=(384, 192, 64)):
    return L.nt_rotary(dtype, B, T, H, D, R, 0, 0, 1.0, x, 384, 192, 64, pos, 2, freq, y, *ys, None)


@pytest.mark.parametrize("bad,status,text", [
    (dict(dtype=2), 2, "dtype"), (dict(R=63), 1, "even"), (dict(R=66), 1, "even"), (dict(R=0), 1, "even"), (dict(B=-1), 1, "sizes"),
    (dict(D=0), 1, "sizes"), (dict(D=2050, R=64), 1, "sizes"), (dict(x=None), 1, "null"), (dict(pos=None), 1, "null"), (dict(freq=None), 1, "null"),
    (dict(y=None), 1, "null"), (dict(ys=(1, 2, 3)), 1, "in place")])
def test_rotary_status(nat, bad, status, text):
    L = nat.load()
    assert rotary(L, **bad) == status
    assert text in L.nt_last_error().decode()


def test_empty_calls_succeed(nat):
    L = nat.load()
    assert rotary(L, B=0, x=None) == 0 and rotary(L, T=0, x=None) == 0
    assert append(L, T=0, k=None) == 0
    assert attention(L, B=0, q=None) == 0
    assert logits(L, B=0, x=None) == 0


def append(L, dtype=1, B=1, T=1, H=2, D=64, page=16, n=4, blocks=2, k=FAKE, codes=FAKE, lengths=FAKE):
    return L.nt_kv_append(dtype, B, T, H, D, page, n, blocks, k, 0, 0, 0, FAKE, 0, 0, 0, codes, FAKE, FAKE, FAKE, FAKE, 2, lengths,
                          None, None)


@pytest.mark.parametrize("bad,status,text", [
    (dict(dtype=2), 2, "dtype"), (dict(D=72), 1, "head_dim"), (dict(page=8), 1, "page"), (dict(page=48), 1, "page"),
    (dict(B=65536), 1, "sizes"), (dict(H=0), 1, "sizes"), (dict(k=None), 1, "null"), (dict(lengths=None), 1, "null"),
    (dict(codes=ctypes.c_void_p(4104)), 1, "alignment")])
def test_append_status(nat, bad, status, text):
    L = nat.load()
    assert append(L, **bad) == status
    assert text in L.nt_last_error().decode()


def attention(L, dtype=1, B=1, T=1, Hq=2, H=2, D=64, page=16, blocks=2, window=-1, q=FAKE, codes=FAKE, ws=None, nbytes=0):
    return L.nt_kv_attention(dtype, B, T, Hq, H, D, page, 4, blocks, window, 1.0, q, 0, 0, 0, codes, FAKE, FAKE, FAKE, FAKE, 2, FAKE,
                             None, FAKE, ws, nbytes, None)


@pytest.mark.parametrize("bad,status,text", [
    (dict(dtype=0x7), 2, "dtype"), (dict(D=256), 1, "head_dim"), (dict(page=128), 1, "page"), (dict(Hq=3), 1, "sizes"),
    (dict(Hq=1), 1, "sizes"), (dict(H=0), 1, "sizes"), (dict(blocks=1 << 28), 1, "sizes"), (dict(q=None), 1, "null"),
    (dict(codes=ctypes.c_void_p(4104)), 1, "alignment"), (dict(blocks=4096), 6, "workspace")])
def test_attention_status(nat, bad, status, text):
    L = nat.load()
    assert attention(L, **bad) == status
    assert text in L.nt_last_error().decode()


def test_attention_workspace_covers_long_caches(nat):
    L = nat.load()
    need = L.nt_kv_attention_workspace_bytes(1, 1, 32, 8, 128, 64, 2048, -1)
    assert need > 0
    assert attention(L, Hq=32, H=8, D=128, page=64, blocks=2048, ws=FAKE, nbytes=need - 1) == 6
    assert L.nt_kv_attention_workspace_bytes(1, 1, 10, 10, 64, 16, 4, -1) == 0        # one CTA per head sees all of it
    assert L.nt_kv_attention_workspace_bytes(0, 1, 1, 1, 64, 16, 4, -1) == 0
    assert L.nt_kv_attention_workspace_bytes(1, 1, 10, 10, 64, 16, 4, 2 ** 63 - 1) == 0


def logits(L, dtype=0, B=1, V=100, x=FAKE, tokens=FAKE, n=5, prompts=None, each=0, rep=1.0, ids=None, nb=0, out=FAKE, ldo=100):
    return L.nt_logits_process(dtype, B, V, x, 100, tokens, 5, n, None, prompts, each, None, rep, None, 0.0, None, 0.0, ids, 0, None, 0,
                               nb, None, 0, out, ldo, None)


@pytest.mark.parametrize("bad,status,text", [
    (dict(dtype=2), 2, "dtype"), (dict(V=0), 1, "sizes"), (dict(B=-1), 1, "sizes"), (dict(x=None), 1, "null"),
    (dict(tokens=None), 1, "null"), (dict(nb=3), 1, "null"), (dict(ldo=101), 1, "in place"), (dict(each=1, prompts=FAKE), 1, "occurrence"),
    (dict(rep=0.0), 1, "above 0"), (dict(rep=float("nan")), 1, "above 0")])
def test_logits_status(nat, bad, status, text):
    L = nat.load()
    assert logits(L, **bad) == status
    assert text in L.nt_last_error().decode()


def test_cpu_tensors_are_refused(nat):
    x = torch.zeros(1, 1, 2, 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.rotary(x, torch.zeros(1, 1, dtype=torch.int64), torch.ones(32))
    c, s = torch.zeros(2, 2, 16, 64, dtype=torch.uint8), torch.ones(2, 2)
    args = (c, s, c.clone(), s.clone(), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.kv_append(x, x, *args)
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.kv_attention(x, *args)
    with pytest.raises(RuntimeError, match="CUDA"):
        nat.logits_process(torch.zeros(1, 10))


def test_pack_allowed_words():
    from neuratensor_b200 import native
    mask = torch.zeros(2, 70, dtype=torch.bool)
    mask[0, [0, 31, 32, 69]] = True
    mask[1] = True
    words = native.pack_allowed(mask)
    assert words.dtype == torch.int32 and words.tolist() == [[-2 ** 31 + 1, 1, 32], [-1, -1, 63]]
    with pytest.raises(ValueError):
        native.pack_allowed(mask.int())


def test_packed_calls_are_the_calls(nat):
    """nt_call_packed reads the arguments in their order: the same refusals, by the argument that is wrong."""
    L = nat.load()

    def call(name, *args):
        entry, n, pack = nat._PACKED[name]
        words = pack(*args)
        assert len(words) == 8 * n
        return L.nt_call_packed(entry, words, n), L.nt_last_error().decode()

    X = 4096
    assert call("nt_rotary", 0, 1, 2, 3, 64, 63, 0, 0, 1.0, X, 1, 2, 3, X, 2, X, X, 1, 2, 3, 0) == (
        1, "nt_rotary: rotated part 63 of 64 must be even, 2..D")
    assert call("nt_rotary", 0, 1, 2, 3, 64, 64, 0, 0, 1.0, X, 1, 2, 3, X, 2, X, X, 1, 2, 4, 0)[1].endswith("equal strides")
    assert call("nt_rotary", 0, 0, 2, 3, 64, 64, 0, 0, 1.0, *[0] * 12)[0] == 0
    assert call("nt_kv_append", 1, 1, 1, 2, 64, 48, 4, 2, *[X] * 17)[1].startswith("nt_kv_append: page of 48 tokens")
    assert call("nt_kv_append", 1, 1, 1, 2, 64, 16, 4, 2, X, 0, 0, 0, X, 0, 0, 0, X, X, X, 0, X, 2, X, 0, 0)[1].endswith("null pointer")
    assert call("nt_kv_append", 1, 1, 0, 2, 64, 16, 4, 2, *[0] * 17)[0] == 0
    args = (1, 1, 1, 32, 8, 128, 64, 4, 2048, -1, 1.0, X, 0, 0, 0, X, X, X, X, X, 2, X, 0, X)
    need = L.nt_kv_attention_workspace_bytes(1, 1, 32, 8, 128, 64, 2048, -1)
    assert call("nt_kv_attention", *args, X, need - 1, 0) == (6, f"nt_kv_attention: workspace {need - 1} < {need} bytes")
    args = (0, 1, 100, X, 100, X, 5, 5, 0, 0, 0, 0, -0.5, 0, 0.0, 0, 0.0, 0, 0, 0, 0, 0, 0, 0, X, 101, 0)
    assert call("nt_logits_process", *args)[1].endswith("in place needs equal row strides")
    args = args[:-2] + (100, 0)
    assert call("nt_logits_process", *args)[1].endswith("must be above 0")
    for entry, words, n, text in ((4, b"", 0, "entry 4"), (-1, b"", 0, "entry -1"), (0, None, 21, "null"), (0, bytes(8), 1, "takes 21")):
        assert L.nt_call_packed(entry, words, n) == 1 and text in L.nt_last_error().decode()


@pytest.mark.parametrize("more,text", [
    (dict(allowed=torch.zeros(1, 70, dtype=torch.bool)), "leaves no token"),
    (dict(allowed=torch.tensor([[True] * 70, [False] * 70])), "leaves no token"),            # of one sequence
    (dict(allowed=torch.tensor([[0, 0, 1 << 6]], dtype=torch.int32)), "leaves no token"),    # a bit behind the vocabulary
    (dict(allowed=torch.cat([torch.zeros(1, 70), torch.ones(1, 26)], 1).bool()), "leaves no token"),
    (dict(allowed=torch.ones(1, 64, dtype=torch.bool)), "allowed must be"),
    (dict(allowed=torch.ones(3, 70, dtype=torch.bool)), "allowed must be"),
    (dict(allowed=torch.ones(1, 70)), "allowed must be"),
    (dict(logit_bias={3: math.inf}), "logit_bias"),
    (dict(logit_bias={3: -math.inf}), "logit_bias"),
    (dict(logit_bias={3: math.nan}), "logit_bias"),
    (dict(logit_bias={70: 1.0}), "logit_bias"),
    (dict(logit_bias={-1: 1.0}), "logit_bias"),
    (dict(frequency_penalty=math.nan), "frequency_penalty"),
    (dict(frequency_penalty=-math.inf), "frequency_penalty"),
    (dict(presence_penalty=math.inf), "presence_penalty"),
    (dict(presence_penalty=1e21), "presence_penalty"),
    (dict(repetition_penalty=0.0), "repetition_penalty"),
    (dict(repetition_penalty=math.nan), "repetition_penalty"),
])
@pytest.mark.parametrize("top_k", [1, 50])
def test_generate_refuses_what_cannot_be_sampled(more, text, top_k):
    """Before anything runs: rows of logits without a finite largest value have no probabilities."""
    from neuratensor_b200 import ModelConfig, NeuraTensorModel
    model = NeuraTensorModel(ModelConfig(vocab_size=70, d_model=128, n_layers=2, d_state=16, max_seq_len=64, attn_every=2,
                                         attn_heads=2, attn_window=8))
    with pytest.raises(ValueError, match=text):
        model.generate(torch.zeros(2, 3, dtype=torch.int64), max_new_tokens=2, top_k=top_k, **more)


def test_allowed_words_of_a_step():
    from neuratensor_b200.core.model import allowed_words
    assert allowed_words(None, 2, 70) is None
    last = torch.zeros(2, 70, dtype=torch.bool)
    last[:, 69] = True
    words = allowed_words(last, 2, 70)
    assert words.tolist() == [[0, 0, 1 << 5]] * 2 and allowed_words(words, 2, 70) is words
    top = torch.zeros(1, 64, dtype=torch.bool)
    top[0, 63] = True                                        # the sign bit of a word
    assert allowed_words(top, 2, 64).tolist() == [[0, -2 ** 31]]
    with pytest.raises(ValueError, match="leaves no token"):
        allowed_words(torch.zeros(2, 3, dtype=torch.int32), 2, 70)


def test_repetition_per_occurrence_takes_what_the_loop_took(nat):
    """v / r and v * r are defined for a negative r.  Every call has prompt lengths, which a penalty per
    occurrence is refused for behind the check of r, so that none launches."""
    L = nat.load()
    for each, r, text in ((0, -1.5, "above 0"), (1, 0.0, "not 0"), (1, math.nan, "not 0"), (1, math.inf, "not 0"),
                          (1, -1.5, "prompt lengths")):
        assert logits(L, each=each, rep=r, prompts=FAKE) == 1
        assert text in L.nt_last_error().decode()
