"""Refusals of pal_paged_attention_chunk (before any launch, so no GPU is needed), its sizing, and the reference itself."""

import math

import pytest
import torch

from chunk_reference import chunk_reference, make_chunk_case


@pytest.fixture(scope="module")
def lib():
    from proxy_attention_lab_b200 import _lib

    return _lib


def _call(lib, **changed):
    a = dict(q=4096, st=512, sh=64, k=4096, v=4096, table=4096, lens=4096, cu=4096, out=4096, seqs=2, total=6, hq=8, hkv=2, d=64, tpp=16,
             pages=10, mp=4, scale=0.0, causal=1, window=0, dtype=1, scratch=4096, scratch_bytes=1 << 40, status=None)
    a.update(changed)
    return lib.lib.pal_paged_attention_chunk(a["q"], a["st"], a["sh"], a["k"], a["v"], a["table"], a["lens"], a["cu"], a["out"], a["seqs"],
                                             a["total"], a["hq"], a["hkv"], a["d"], a["tpp"], a["pages"], a["mp"], a["scale"], a["causal"],
                                             a["window"], a["dtype"], a["scratch"], a["scratch_bytes"], a["status"], None)


def test_arguments(lib):
    assert _call(lib, total=0) == lib.PAL_OK and _call(lib, seqs=0) == lib.PAL_OK
    for changed in (dict(seqs=-1), dict(total=-1), dict(pages=-1), dict(mp=-1), dict(hq=7), dict(hkv=0), dict(d=0), dict(window=-1),
                    dict(window=3, causal=0), dict(q=None), dict(out=None), dict(lens=None), dict(k=None), dict(table=None), dict(q=4104),
                    dict(v=4100), dict(st=516), dict(sh=4), dict(cu=None, total=5), dict(total=1 << 31), dict(st=-8), dict(st=1 << 40)):
        assert _call(lib, **changed) == lib.PAL_ERR_BAD_ARG, changed
        assert "paged_attention_chunk" in lib.last_error()
    for changed in (dict(dtype=2), dict(dtype=2 | lib.PAL_OUT_F32), dict(pages=1 << 31)):
        assert _call(lib, **changed) == lib.PAL_ERR_UNSUPPORTED, changed
    for changed in (dict(d=48), dict(tpp=8)):
        assert _call(lib, **changed) == lib.PAL_ERR_UNSUPPORTED, changed
        assert "no kernel" in lib.last_error()
    for changed in (dict(scratch=None), dict(scratch=4097), dict(scratch_bytes=16)):
        assert _call(lib, **changed) == lib.PAL_ERR_WORKSPACE, changed


def test_scratch_follows_the_shape(lib):
    f = lib.lib.pal_chunk_scratch_bytes
    assert f(0, 8, 2, 64) == 0 and f(5, 7, 2, 64) == 0
    # two partial slots per CTA, a row of D + 2 floats for every row an item can have
    assert f(1, 32, 8, 128) >= 2 * 148 * 4 * (128 + 2) * 4
    assert f(10 ** 6, 32, 8, 128) == f(64, 32, 8, 128) >= 2 * 148 * 256 * (128 + 2) * 4
    assert f(10 ** 6, 32, 8, 256) < f(10 ** 6, 32, 8, 128) * 1.1  # one accumulator tile


def test_cpu_tensors_are_rejected():
    import proxy_attention_lab_b200 as pal

    case = make_chunk_case(0, [1], [4], 2, 1, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pal.paged_attention_chunk(case["q"], case["k_pool"], case["v_pool"], case["table"], case["lens"], case["cu"])


@pytest.mark.parametrize("causal,window", [(True, None), (True, 20), (False, None)])
def test_reference_against_dense_attention(causal, window):
    """The definition through the pages equals masked dense attention (a different route to the same keys)."""
    new, lens, hq, hkv, d = [5, 1, 33], [40, 9, 33], 4, 2, 64
    case = make_chunk_case(3, new, lens, hq, hkv, d, window=window)
    out, bound = chunk_reference(case, causal)
    assert (bound >= 0).all()
    row = 0
    for s, (n, L) in enumerate(zip(new, lens)):
        ids = case["table"][s].long().clamp(min=0)[:-(-L // 16)]
        k = case["k_pool"][ids].permute(0, 3, 1, 2, 4).reshape(-1, hkv, d)[:L].double()
        v = case["v_pool"][ids].permute(0, 3, 1, 2).reshape(-1, hkv, d)[:L].double()
        for i in range(n):
            pos = L - n + i
            a = max(0, pos - window + 1) if window else 0
            b = pos + 1 if causal else L
            for h in range(hq):
                p = torch.softmax(k[a:b, h // 2] @ case["q"][row + i, h].double() / math.sqrt(d), 0)
                assert torch.allclose(out[row + i, h], p @ v[a:b, h // 2])
        row += n
