"""Serving operators without a GPU: the C entries' refusals, the structures' layout, the rotary tables."""
import math

import pytest
import torch

from dpuf_b200 import _native, engine, serving

ADDR = 1 << 20  # a 16-byte aligned stand-in for device memory: refused calls never touch it


@pytest.fixture(scope="module")
def lib():
    _native.build_cuda()
    return serving._lib()


def kv(**over):
    a = dict(k=ADDR, v=ADDR, page=16 * 2 * 64, head=16 * 64, row=64, dtype=1, n_pages=4, n_kv=2, size=16, dim=64)
    a.update(over)
    return serving._KV.pack(a["k"], a["v"], a["page"], a["head"], a["row"], a["dtype"], a["n_pages"], a["n_kv"],
                            a["size"], a["dim"], 0)


def rope_args(cache=None, **over):
    a = dict(table=ADDR, tstride=4, q=ADDR, k=ADDR, v=ADDR, out=ADDR, cos=ADDR, sin=ADDR, seq=ADDR, pos=ADDR, seqs=1,
             width=4, n=1, n_q=4, rot=64, n_pos=64, inter=0, dtype=1, odtype=1)
    a.update(over)
    return (cache or kv()) + serving._ROPE.pack(a["table"], a["tstride"], a["q"], a["k"], a["v"], 256, 64, 128, 64,
                                                128, 64, a["out"], a["cos"], a["sin"], a["seq"], a["pos"], a["seqs"],
                                                a["width"], a["n"], a["n_q"], a["rot"], a["n_pos"], a["inter"],
                                                a["dtype"], a["odtype"], 0)


def attn_args(cache=None, **over):
    a = dict(table=ADDR, tstride=4, q=ADDR, qs0=256, qs1=64, out=ADDR, q_start=ADDR, kv_len=ADDR, ws=ADDR,
             ws_bytes=1 << 40, seqs=1, width=4, n=1, n_q=4, max_q=1, causal=1, window=0, dtype=1, odtype=1, scale=0.125)
    a.update(over)
    return (cache or kv()) + serving._ATTN.pack(a["table"], a["tstride"], a["q"], a["qs0"], a["qs1"], a["out"],
                                                a["q_start"], a["kv_len"], a["ws"], a["ws_bytes"], a["seqs"],
                                                a["width"], a["n"], a["n_q"], a["max_q"], a["causal"], a["window"],
                                                a["dtype"], a["odtype"], a["scale"])


BAD_CACHE = [dict(k=0), dict(v=0), dict(k=ADDR + 8), dict(dtype=3), dict(dtype=-1), dict(n_pages=0), dict(n_kv=0),
             dict(size=4), dict(size=24), dict(size=2048), dict(dim=0), dict(dim=60), dict(dim=264), dict(row=63),
             dict(row=68), dict(head=1028), dict(page=-2048)]


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_caches_are_refused(lib, bad):
    assert lib.dpuf_cuda_rope_append(rope_args(kv(**bad)), None) == -1
    assert engine.last_error().startswith("dpuf_cuda_rope_append: ")
    assert lib.dpuf_cuda_paged_attention(attn_args(kv(**bad)), None) == -1
    assert engine.last_error().startswith("dpuf_cuda_paged_attention: ")


@pytest.mark.parametrize("bad", [dict(table=0), dict(tstride=3), dict(seqs=0), dict(width=0), dict(n=-1), dict(q=0),
                                 dict(k=0), dict(v=0), dict(out=0), dict(cos=0), dict(sin=0), dict(seq=0), dict(pos=0),
                                 dict(n_q=0), dict(rot=0), dict(rot=63), dict(rot=66), dict(n_pos=0), dict(dtype=7),
                                 dict(odtype=-1)], ids=str)
def test_rope_append_refusals(lib, bad):
    assert lib.dpuf_cuda_rope_append(rope_args(**bad), None) == -1
    assert engine.last_error()


@pytest.mark.parametrize("bad", [dict(table=0), dict(tstride=3), dict(seqs=0), dict(n=-1), dict(q=0), dict(out=0),
                                 dict(q_start=0), dict(kv_len=0), dict(ws=0), dict(ws=ADDR + 4), dict(ws_bytes=64),
                                 dict(n_q=3), dict(n_q=0), dict(max_q=0), dict(max_q=1 << 30), dict(window=-1),
                                 dict(window=4, causal=0), dict(dtype=2), dict(odtype=2), dict(scale=math.inf),
                                 dict(scale=math.nan), dict(q=ADDR + 2), dict(qs0=257), dict(qs1=60)], ids=str)
def test_paged_attention_refusals(lib, bad):
    assert lib.dpuf_cuda_paged_attention(attn_args(**bad), None) == -1
    assert engine.last_error()


@pytest.mark.parametrize("bad", [dict(logits=0), dict(logits=ADDR + 2), dict(dtype=5), dict(rows=-1), dict(vocab=0),
                                 dict(vocab=(1 << 20) + 1), dict(u=0), dict(ids=0)], ids=str)
def test_sample_refusals(lib, bad):
    a = dict(logits=ADDR, dtype=0, stride=8, rows=1, vocab=8, u=ADDR, ids=ADDR)
    a.update(bad)
    assert lib.dpuf_cuda_sample_rows(a["logits"], a["dtype"], a["stride"], a["rows"], a["vocab"], a["u"], None, None,
                                     None, None, a["ids"], None, None) == -1
    assert engine.last_error().startswith("dpuf_cuda_sample_rows: ")


def test_empty_calls_do_nothing(lib):
    assert lib.dpuf_cuda_rope_append(rope_args(n=0), None) == 0
    assert lib.dpuf_cuda_paged_attention(attn_args(n=0), None) == 0
    assert lib.dpuf_cuda_sample_rows(ADDR, 0, 8, 0, 8, ADDR, None, None, None, None, ADDR, None, None) == 0
    assert engine.last_error() == ""
    for fn in (lib.dpuf_cuda_rope_append, lib.dpuf_cuda_paged_attention, lib.dpuf_cuda_paged_attention_status):
        assert fn(None, None) == -1


def test_a_batch_of_no_sequences_does_nothing(lib):
    """No tokens of no sequences: a table of no rows or no entries, whose tensor has no address."""
    for over in (dict(seqs=0), dict(width=0, tstride=0), dict(seqs=0, width=0, tstride=0)):
        assert lib.dpuf_cuda_rope_append(rope_args(n=0, table=0, **over), None) == 0
        assert lib.dpuf_cuda_paged_attention(attn_args(n=0, table=0, **over), None) == 0
        assert lib.dpuf_cuda_rope_append(rope_args(kv(n_kv=0), n=0, table=0, **over), None) == -1
        assert lib.dpuf_cuda_paged_attention(attn_args(kv(n_kv=0), n=0, table=0, **over), None) == -1
    assert lib.dpuf_cuda_rope_append(rope_args(n=0, table=0, seqs=-1), None) == -1
    assert lib.dpuf_cuda_paged_attention(attn_args(n=0, table=0, width=-1), None) == -1


def test_cache_refuses_host_tensors():
    x = torch.zeros(2, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        serving.PagedCache(x, x)
    with pytest.raises(TypeError):
        serving.PagedCache(x.double(), x.double())


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn", "llama3"])
@pytest.mark.parametrize("rot", [2, 10, 64])
def test_rope_table(scaling, rot):
    if scaling == "ntk" and rot == 2:
        with pytest.raises(ValueError):
            serving.rope_table(8, rot, scaling=scaling, factor=2.0, device="cpu")
        return
    theta, factor, orig, n = 1e4, 4.0, 512, 2048
    cos, sin = serving.rope_table(n, rot, theta, scaling, factor, orig, device="cpu")
    assert cos.shape == sin.shape == (n, rot // 2) and cos.dtype == torch.float32
    for i in range(rot // 2):
        f = theta ** (-2 * i / rot)
        gain = 1.0
        if scaling == "linear":
            f /= factor
        elif scaling == "ntk":
            f = (theta * factor ** (rot / (rot - 2))) ** (-2 * i / rot)
        elif scaling == "yarn":
            turns = orig * f / (2 * math.pi)
            ramp = min(1.0, max(0.0, (turns - 1) / 31))
            f = f * ramp + f / factor * (1 - ramp)
            gain = 0.1 * math.log(factor) + 1
        elif scaling == "llama3":
            wave = 2 * math.pi / f
            if wave > orig:
                f /= factor
            elif wave > orig / 4:
                mix = (orig / wave - 1) / 3
                f = (1 - mix) * f / factor + mix * f
        for p in (0, 1, 77, n - 1):
            # one rounding to float32 of a value up to `gain`, and the angle's error in 64 bits
            tol = gain * 2.0 ** -24 + p * f * 1e-15
            assert abs(float(cos[p, i]) - gain * math.cos(p * f)) <= tol
            assert abs(float(sin[p, i]) - gain * math.sin(p * f)) <= tol


@pytest.mark.parametrize("args", [dict(rotary_dim=3), dict(rotary_dim=0), dict(n_pos=0), dict(factor=0.0),
                                  dict(scaling="yarn"), dict(scaling="llama3"), dict(scaling="other")], ids=str)
def test_rope_table_refusals(args):
    a = dict(n_pos=8, rotary_dim=8, device="cpu")
    a.update(args)
    with pytest.raises(ValueError):
        serving.rope_table(**a)
