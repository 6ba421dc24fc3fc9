"""Refusals of the rotary entry points of the C ABI (all before any launch, so no GPU is needed), and the reference itself."""

import ctypes

import pytest
import torch

from rotary_reference import axis_of_frequency, rotate64


@pytest.fixture(scope="module")
def lib():
    from proxy_attention_lab_b200 import _lib

    return _lib


def _rotation(lib, **changed):
    dummy = ctypes.create_string_buffer(64)
    fields = dict(positions=ctypes.addressof(dummy), positions_axis_stride=0, inv_freq=ctypes.addressof(dummy), magnitude=1.0, num_freqs=8,
                  num_axes=1, sections=(0, 0, 0, 0), section_order=0, pairing=0, positions_64bit=0)
    fields.update(changed)
    fields["sections"] = (ctypes.c_int32 * 4)(*fields["sections"])
    rot = lib.Rotation(**fields)
    rot.keep = dummy
    return rot


def _rotate(lib, rot, tokens=0, heads=1, d=16, dtype=0, x=None, out=None):
    return lib.lib.pal_rotary_embedding(x, out, rot, tokens, heads, d, dtype, None)


def test_rotation_arguments(lib):
    assert _rotate(lib, _rotation(lib)) == lib.PAL_OK  # no tokens: nothing to launch
    assert _rotate(lib, _rotation(lib), tokens=3, heads=0) == lib.PAL_OK
    assert _rotate(lib, _rotation(lib), dtype=3) == lib.PAL_ERR_UNSUPPORTED
    for changed in (dict(num_freqs=0), dict(num_freqs=9), dict(num_axes=0), dict(num_axes=5), dict(pairing=2), dict(section_order=-1),
                    dict(inv_freq=None), dict(num_axes=2, sections=(4, 3, 0, 0)), dict(num_axes=2, sections=(9, -1, 0, 0)),
                    dict(num_axes=2, sections=(2, 6, 0, 0), section_order=1)):
        assert _rotate(lib, _rotation(lib, **changed)) == lib.PAL_ERR_BAD_ARG, changed
        assert "rotary_embedding" in lib.last_error()
    assert _rotate(lib, None) == lib.PAL_ERR_BAD_ARG
    assert _rotate(lib, _rotation(lib), tokens=-1) == lib.PAL_ERR_BAD_ARG
    assert _rotate(lib, _rotation(lib), d=0) == lib.PAL_ERR_BAD_ARG
    assert _rotate(lib, _rotation(lib), tokens=1) == lib.PAL_ERR_BAD_ARG  # x is null
    assert _rotate(lib, _rotation(lib, positions=None), tokens=1) == lib.PAL_ERR_BAD_ARG
    rows = lib.Rows(3, 16, 16)  # an odd address
    assert _rotate(lib, _rotation(lib), tokens=1, x=rows, out=rows) == lib.PAL_ERR_BAD_ARG
    assert _rotate(lib, _rotation(lib, num_axes=3, sections=(3, 3, 2, 0), section_order=1)) == lib.PAL_OK


def test_append_arguments(lib):
    rows = lib.Rows(4096, 32, 16)

    def call(k=rows, v=rows, q=None, qo=None, pools=4096, slots=4096, table=None, wp=None, sm=None, rot=_rotation(lib), tokens=1, seqs=0, hq=0,
             hkv=1, d=16, tpp=16, pages=1, mp=0, dtype=0):
        return lib.lib.pal_fill_kv_pages_rotary(k, v, q, qo, pools, pools, slots, table, wp, sm, rot, tokens, seqs, hq, hkv, d, tpp, pages, mp, dtype,
                                                None)

    assert call(tokens=0) == lib.PAL_OK
    assert call(dtype=2) == lib.PAL_ERR_UNSUPPORTED
    assert call(d=20) == lib.PAL_ERR_UNSUPPORTED and call(d=264) == lib.PAL_ERR_UNSUPPORTED
    for changed in (dict(k=None), dict(v=lib.Rows(None, 1, 1)), dict(hq=2), dict(hq=-1), dict(hkv=0), dict(tpp=0), dict(pages=-1), dict(tokens=-1),
                    dict(pools=None), dict(pools=4104), dict(slots=None, mp=1), dict(slots=None, table=4096, wp=4096, mp=1), dict(rot=None),
                    dict(k=lib.Rows(4097, 1, 1))):
        assert call(**changed) == lib.PAL_ERR_BAD_ARG, changed
        assert "fill_kv_pages_rotary" in lib.last_error()


def test_append_addresses_are_required_whatever_the_tables_width(lib):
    """Without slots the positions and sequences of the tokens are read even when the page table is empty: null ones are refused
    before a launch."""
    rows, rot = lib.Rows(4096, 32, 16), _rotation(lib)
    for mp, seqs in ((0, 0), (0, 3), (4, 0), (4, 3)):
        for wp, sm in ((None, None), (4096, None), (None, 4096)):
            rc = lib.lib.pal_fill_kv_pages_rotary(rows, rows, None, None, 4096, 4096, None, 4096, wp, sm, rot, 1, seqs, 0, 1, 16, 16, 1, mp, 0, None)
            assert rc == lib.PAL_ERR_BAD_ARG, (mp, seqs, wp, sm)
            assert "are required" in lib.last_error()


def test_cpu_tensors_are_rejected():
    import proxy_attention_lab_b200 as pal

    x = torch.zeros((1, 2, 64), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pal.rotary_embedding(x, torch.zeros(1, dtype=torch.int32), torch.ones(32))
    k = torch.zeros((1, 2, 8, 16, 8), dtype=torch.float16)
    v = torch.zeros((1, 2, 64, 16), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pal.fill_kv_pages_rotary(x, x, k, v, torch.zeros(1, dtype=torch.int64), inv_freq=torch.ones(32), positions=torch.zeros(1))


def test_reference_is_a_rotation():
    g = torch.Generator().manual_seed(0)
    x = torch.randn((6, 2, 32), generator=g, dtype=torch.float64)
    pos = torch.randint(0, 1000, (3, 6), generator=g)
    freq = torch.rand(12, generator=g)
    for order, sections in (("blocked", [4, 5, 3]), ("interleaved", [5, 4, 3])):
        assert sorted(axis_of_frequency(12, sections, order)) == [a for a, n in enumerate(sections) for _ in range(n)]
        for pairing in ("half", "adjacent"):
            y = rotate64(x, pos, freq, sections, order, pairing)
            assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1))
            assert torch.allclose(rotate64(y, -pos, freq, sections, order, pairing), x)
    assert axis_of_frequency(8, [4, 2, 2], "interleaved") == [0, 1, 2, 0, 1, 2, 0, 0]
    # scores of rotated queries and keys depend on the difference of their positions alone
    q, k = x[:1], x[1:2]
    one = lambda a, b: (rotate64(q, torch.tensor([a]), freq) * rotate64(k, torch.tensor([b]), freq)).sum()
    assert torch.allclose(one(10, 3), one(1010, 1003))
