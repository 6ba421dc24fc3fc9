"""paged_attention_chunk against the definition in 64 bits."""

import sys

import pytest
import torch

from chunk_reference import assert_chunk, make_chunk_case

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def short_waits(pal, cuda):
    """A wait that cannot end gives up after a quarter of a second and fails the test."""
    from proxy_attention_lab_b200 import _lib

    before = _lib.lib.pal_set_wait_limit_cycles(500_000_000)
    yield
    torch.cuda.synchronize()
    pal.check_status()
    _lib.lib.pal_set_wait_limit_cycles(before)


def _run(pal, case, **kw):
    return pal.paged_attention_chunk(case["q"], case["k_pool"], case["v_pool"], case["table"], case["lens"], case["cu"],
                                     window=case["window"], **kw)


SHAPES = [
    # (new tokens, lengths, hq, hkv)
    ([1], [1], 1, 1),
    ([1], [128], 4, 1),
    ([1], [129], 4, 1),
    ([5], [1000], 32, 8),
    ([5, 1, 3, 9], [5, 700, 3, 40], 8, 2),
    ([200], [200], 4, 2),
    ([64, 65, 33, 1, 128], [64, 300, 33, 77, 1000], 4, 1),
    ([300, 1, 0, 129], [700, 513, 40, 129], 6, 2),     # three heads per kv head: 126 of 128 rows used
    ([257], [2049], 2, 2),                            # one head per kv head
    ([40, 7], [90, 2000], 14, 2),                     # seven
    ([3, 70], [500, 70], 40, 1),                      # forty: three tokens per tile
    ([2, 5], [300, 5], 150, 1),                       # more heads than a tile has rows
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("new,lens,hq,hkv", SHAPES)
def test_shapes(pal, cuda, new, lens, hq, hkv, dtype):
    case = make_chunk_case(sum(lens), new, lens, hq, hkv, 128, dtype=dtype, device=cuda)
    out = _run(pal, case)
    assert out.shape == case["q"].shape and out.dtype == dtype
    assert_chunk(out, case)


@pytest.mark.parametrize("tpp", [16, 32])
@pytest.mark.parametrize("d", [32, 64, 80, 96, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_every_instantiation(pal, cuda, d, tpp, dtype):
    case = make_chunk_case(d + tpp, [150, 4, 1, 33], [600, 333, 1500, 33], 6, 2, d, tpp=tpp, dtype=dtype, device=cuda)
    assert_chunk(_run(pal, case), case)


@pytest.mark.parametrize("d,hq,hkv", [(128, 8, 2), (64, 3, 1), (256, 4, 2)])
def test_float32_output(pal, cuda, d, hq, hkv):
    case = make_chunk_case(7, [90, 2], [400, 900], hq, hkv, d, dtype=BF16, device=cuda)
    out = _run(pal, case, out_dtype=torch.float32)
    assert out.dtype == torch.float32
    assert_chunk(out, dict(case, out_dtype=torch.float32))


@pytest.mark.parametrize("window", [1, 16, 100, 128, 500, 5000])
@pytest.mark.parametrize("d,tpp", [(128, 16), (64, 32), (256, 16)])
def test_window(pal, cuda, window, d, tpp):
    case = make_chunk_case(window, [180, 1, 5, 64], [700, 900, 130, 64], 8, 2, d, tpp=tpp, dtype=BF16, device=cuda, window=window)
    assert_chunk(_run(pal, case), case)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, sys.maxsize, 2 ** 80])
@pytest.mark.parametrize("stream", [False, True])
def test_windows_wider_than_any_sequence(pal, cuda, window, stream):
    """A window past 32 bits, which is a usual way to say that there is none, through either front."""
    case = make_chunk_case(5, [40, 1, 9, 70], [90, 700, 4, 0], 8, 2, 128, dtype=BF16, device=cuda)
    plain = _run(pal, case).clone()
    kw = dict(stream=torch.cuda.current_stream()) if stream else {}
    out = pal.paged_attention_chunk(case["q"], case["k_pool"], case["v_pool"], case["table"], case["lens"], case["cu"], window=window, **kw)
    assert torch.equal(out.view(torch.int16), plain.view(torch.int16))


@pytest.mark.parametrize("d", [128, 256, 32])
def test_all_keys(pal, cuda, d):
    case = make_chunk_case(11, [70, 1, 300], [70, 900, 555], 4, 2, d, dtype=FP16, device=cuda)
    assert_chunk(_run(pal, case, causal=False), case, causal=False)


def test_rows_without_keys_are_zero(pal, cuda):
    """Lengths of zero, and lengths below the number of rows: the first rows stand before the sequence."""
    case = make_chunk_case(12, [4, 1, 70, 3], [0, 0, 20, 1], 4, 2, 128, dtype=BF16, device=cuda)
    out = _run(pal, case)
    assert_chunk(out, case)
    assert not out[:5].any() and not out[5:5 + 50].any() and out[55:75].any()


@pytest.mark.parametrize("d,tpp", [(32, 32), (64, 16), (64, 32), (80, 16), (128, 16), (256, 16)])
@pytest.mark.parametrize("out_dtype", [None, torch.float32])
def test_rows_without_keys_leave_their_neighbours_alone(pal, cuda, d, tpp, out_dtype):
    """Sequences without keys, of rows for two row tiles, each before a short one whose key tiles (three, or six) are shared by the
    two accumulators: the zeros of the former go out while the latter's accumulators meet."""
    for new, lens, hq, hkv in (([64, 1] * 64, [0, 300] * 64, 32, 8), ([64, 4] * 32, [0, 300] * 32, 32, 8), ([300, 2] * 40, [0, 700] * 40, 8, 2)):
        case = make_chunk_case(d + len(new), new, lens, hq, hkv, d, tpp=tpp, dtype=BF16, device=cuda)
        case["out_dtype"] = out_dtype
        empty = torch.cat([torch.full((n,), L == 0) for n, L in zip(new, lens)]).to(cuda)
        for _ in range(3):
            out = _run(pal, case, out_dtype=out_dtype)
            assert_chunk(out, case)
            assert not out[empty].any()


def test_no_pages_and_no_rows(pal, cuda):
    q = torch.randn((3, 4, 128), device=cuda).to(BF16)
    k = torch.empty((0, 2, 16, 16, 8), dtype=BF16, device=cuda)
    v = torch.empty((0, 2, 128, 16), dtype=BF16, device=cuda)
    lens = torch.full((3,), 5, dtype=torch.int32, device=cuda)
    assert not pal.paged_attention_chunk(q, k, v, torch.zeros((3, 2), dtype=torch.int32, device=cuda), lens).any()
    assert not pal.paged_attention_chunk(q, k, v, torch.zeros((3, 0), dtype=torch.int32, device=cuda), lens).any()
    assert pal.paged_attention_chunk(q[:0], k, v, torch.zeros((3, 2), dtype=torch.int32, device=cuda), lens).shape == (0, 4, 128)
    empty = torch.zeros((0, 2), dtype=torch.int32, device=cuda)
    assert pal.paged_attention_chunk(q[:0], k, v, empty, lens[:0]).shape == (0, 4, 128)


@pytest.mark.parametrize("new,lens", [([1], [60000]), ([7], [33000]), ([1] * 3, [20000, 3, 11000]), ([200], [9000])])
def test_long_sequences_are_cut(pal, cuda, new, lens):
    case = make_chunk_case(13, new, lens, 8, 1, 128, dtype=BF16, device=cuda)
    assert_chunk(_run(pal, case), case)


def test_many_short_sequences(pal, cuda):
    g = torch.Generator().manual_seed(14)
    lens = torch.randint(1, 200, (700,), generator=g).tolist()
    new = [min(L, int(n)) for L, n in zip(lens, torch.randint(0, 5, (700,), generator=g))]
    case = make_chunk_case(14, new, lens, 4, 2, 64, dtype=FP16, device=cuda)
    assert_chunk(_run(pal, case), case)


@pytest.mark.parametrize("d,tpp", [(32, 16), (64, 16), (64, 32), (96, 32), (128, 16)])
@pytest.mark.parametrize("hq,hkv", [(32, 8), (12, 4), (16, 16)])
def test_items_of_one_and_two_row_tiles_in_turn(pal, cuda, d, tpp, hq, hkv):
    """Rows that fill one tile or part of it (their two accumulators are merged in the second query tile's place) between items
    of two tiles, of one, two and more key tiles: a tile of queries is not loaded before the merge in its place has been read."""
    g = torch.Generator().manual_seed(d + hq)
    pick = lambda values, n: [values[int(i)] for i in torch.randint(0, len(values), (n,), generator=g)]
    for dtype in (BF16, FP16):
        new = pick([1, 1, 5, 20, 91, 130, 260], 48)
        lens = [n + h for n, h in zip(new, pick([0, 17, 130, 260, 900], 48))]
        case = make_chunk_case(d, new, lens, hq, hkv, d, tpp=tpp, dtype=dtype, device=cuda)
        for _ in range(4):
            assert_chunk(_run(pal, case), case)


SHORT_ROWS = [
    # (new tokens, lengths, window, causal)
    ([1] * 40, [2, 4, 8, 16] * 10, None, True),        # decode steps at the start of their sequences
    ([1] * 24, [33, 64, 128, 255, 300, 700] * 4, None, True),
    ([5, 9, 16, 3] * 4, [5, 20, 18, 255] * 4, None, True),
    ([300, 70], [300, 90], None, True),                # prompts: their first rows see few keys
    ([1, 3, 200] * 3, [900, 500, 700] * 3, 7, True),   # small windows
    ([4, 1, 150] * 3, [4, 9, 200] * 3, None, False),
]


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (16, 16, 64), (8, 2, 256)])
@pytest.mark.parametrize("new,lens,window,causal", SHORT_ROWS)
def test_short_rows_keep_to_the_parity_rule(pal, cuda, new, lens, window, causal, hq, hkv, d):
    """The rule of the decode and prefill operators, element by element: bf16 outputs within 2e-3, or one unit in the last place, of
    the result, for rows whose few keys average nothing out.

    The residual of P leaves relative errors of at most 2^-16 of a weight, so that an output in fp32 is within 2^-16 (A + |out|) of the
    result (A = sum p |v|, at most 6 over these draws): 2e-4, and rounded one unit in the last place away at most wherever 2e-3 is
    less than a unit.  Rows of 256 keys and more in prompts have a standard deviation of 2^-9 / sqrt(3) * sqrt(sum p^2) * |v| =
    1.1e-3 * 0.1 * 1 of their result: 2e-3 is 18 of them."""
    from cases import assert_parity
    from chunk_reference import chunk_reference

    case = make_chunk_case(sum(lens) + d, new, lens, hq, hkv, d, dtype=BF16, device=cuda, window=window)
    ref, _ = chunk_reference(case, causal)
    assert_parity(_run(pal, case, causal=causal), ref)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 200])
def test_small_weights_of_half_precision_count(pal, cuda, d, new):
    """One key of a tile takes the weight, with value 0; each other one has exp(-18) = 2^-26 of it and value 1.

    Weights are held times 2^7 in steps of 2^-24: each off by at most 2^-32 of the largest, 127 to a tile, beside the errors of the
    exponential (D 2^-24 * 18 * 2 + 2^-22 relative)."""
    hkv, length, tpp = 2, 2048, 16
    pages = length // tpp
    k = torch.zeros((pages, hkv, d // 8, tpp, 8), dtype=FP16, device=cuda)
    v = torch.ones((pages, hkv, d, tpp), dtype=FP16, device=cuda)
    k[::8, :, :, 0] = 1.5   # tokens 0, 128, 256, ...
    v[::8, :, :, 0] = 0.0
    q = torch.full((new, 4, d), 1.5, dtype=FP16, device=cuda)
    table = torch.arange(pages, dtype=torch.int32, device=cuda)[None]
    lens = torch.tensor([length], dtype=torch.int32, device=cuda)
    out = pal.paged_attention_chunk(q, k, v, table, lens, scale=8.0 / d, out_dtype=torch.float32).double()
    seen = torch.arange(length - new, length, device=cuda) + 1
    large = (seen + 127) // 128
    w = torch.exp(torch.tensor(-18.0, dtype=torch.float64))
    ref = ((seen - large) * w / (large + (seen - large) * w))[:, None, None]
    assert ((out - ref).abs() <= 127 * 2.0 ** -32 + (36 * d * 2.0 ** -24 + 2.0 ** -22) * ref).all()


def test_scale_and_large_scores(pal, cuda):
    """Scores of hundreds: the running maximum moves, and single keys take all the weight."""
    case = make_chunk_case(15, [100, 2], [800, 1500], 8, 2, 128, dtype=BF16, device=cuda, q_scale=20.0)
    assert_chunk(_run(pal, case), case)
    assert_chunk(_run(pal, case, scale=0.5), case, scale=0.5)


def test_uniform_batches_need_no_offsets(pal, cuda):
    case = make_chunk_case(16, [6] * 5, [6, 90, 300, 17, 1000], 8, 2, 128, dtype=BF16, device=cuda)
    a = pal.paged_attention_chunk(case["q"], case["k_pool"], case["v_pool"], case["table"], case["lens"])
    assert torch.equal(a.view(torch.int16), _run(pal, case).view(torch.int16))
    assert_chunk(a, case)


def test_rows_behind_the_last_sequence_stay(pal, cuda):
    case = make_chunk_case(17, [5, 40], [50, 400], 4, 2, 128, dtype=BF16, device=cuda, extra_rows=9)
    out = torch.full_like(case["q"], 7.0)
    got = _run(pal, case, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (out[45:] == 7.0).all()
    assert_chunk(out, case)


@pytest.mark.parametrize("kind", ["slice", "offset", "head_major", "int64"])
def test_strided_queries_and_index_types(pal, cuda, kind):
    case = make_chunk_case(18, [30, 2], [200, 90], 8, 2, 64, dtype=FP16, device=cuda)
    q = case["q"]
    if kind == "slice":
        wide = torch.zeros((32, 12, 64), dtype=FP16, device=cuda)
        wide[:, 2:10] = q
        case["q"] = wide[:, 2:10]
    elif kind == "offset":  # not 16-byte aligned: copied
        flat = torch.zeros(q.numel() + 1, dtype=FP16, device=cuda)
        flat[1:] = q.flatten()
        case["q"] = flat[1:].view(q.shape)
    elif kind == "head_major":
        case["q"] = q.transpose(0, 1).contiguous().transpose(0, 1)
    else:
        for name in ("table", "lens", "cu"):
            case[name] = case[name].long()
    out = _run(pal, case)
    assert out.is_contiguous()
    assert_chunk(out, case)


def test_repeated_calls_agree_bit_for_bit(pal, cuda):
    case = make_chunk_case(19, [1, 300, 8, 1], [5000, 900, 2000, 64], 16, 4, 128, dtype=BF16, device=cuda)
    first = _run(pal, case).clone()
    for _ in range(5):
        assert torch.equal(_run(pal, case).view(torch.int16), first.view(torch.int16))


@pytest.mark.parametrize("d,tpp", [(32, 16), (64, 32), (128, 16), (256, 16)])
@pytest.mark.parametrize("hq,hkv", [(12, 4), (14, 2), (8, 8)])
def test_rows_of_a_tile_that_do_not_exist_change_nothing(pal, cuda, d, tpp, hq, hkv):
    """Three heads per kv head leave two rows of a tile unused, seven leave two, and short items more: bit for bit the same
    results whatever stands there, and whatever the calls before left in shared memory."""
    new, lens = [260, 91, 130, 5, 43] * 8, [1160, 91, 260, 400, 43] * 8
    case = make_chunk_case(d, new, lens, hq, hkv, d, tpp=tpp, dtype=BF16, device=cuda)
    other = make_chunk_case(d + 1, [200] * 64, [300] * 64, hq, hkv, d, tpp=tpp, dtype=BF16, device=cuda, q_scale=50.0)
    out = _run(pal, case).clone()
    for _ in range(6):
        _run(pal, other)
        assert torch.equal(out, _run(pal, case))


def test_agrees_with_decode_and_prefill(pal, cuda):
    """One token per sequence is the decode step; a chunk is the prefill with the same keys appended first."""
    case = make_chunk_case(20, [1] * 6, [300, 1, 2000, 17, 128, 900], 32, 8, 128, dtype=BF16, device=cuda)
    a = _run(pal, case).float()
    b = pal.paged_attention_decode(case["q"], case["k_pool"], case["v_pool"], case["table"], case["lens"]).float()
    # both round P and the output to bf16: |a - b| <= 2 (eps / 2) (|v| + |out|) with |v| <= 5 over these draws
    assert (a - b).abs().max() <= 2.0 ** -8 * 10
    new, hist, hq, hkv, d, tpp = 70, 45, 8, 2, 128, 16
    case = make_chunk_case(21, [new], [new + hist], hq, hkv, d, dtype=BF16, device=cuda)
    tok = torch.arange(hist, hist + new, device=cuda)
    page = case["table"][0].long()[tok // tpp]
    kn = case["k_pool"][page, :, :, tok % tpp].reshape(new, hkv, d).contiguous()
    vn = case["v_pool"][page, :, :, tok % tpp].contiguous()
    c = pal.paged_attention_prefill(case["q"], kn, vn, case["k_pool"], case["v_pool"], case["table"],
                                    torch.tensor([hist], dtype=torch.int32, device=cuda)).view(new, hq, d).float()
    assert (_run(pal, case).float() - c).abs().max() <= 2.0 ** -8 * 10


def test_two_streams_at_once(pal, cuda):
    cases = [make_chunk_case(22 + i, [1, 50], [8000, 3000 + i], 8, 2, 128, dtype=BF16, device=cuda) for i in range(2)]
    alone = [_run(pal, c).clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(4):
        outs = [_run(pal, c, stream=s) for c, s in zip(cases, streams)]
        torch.cuda.synchronize()
        for a, b in zip(outs, alone):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_two_graphs_replayed_at_once(pal, cuda):
    cases = [make_chunk_case(24 + i, [1, 50], [8000, 3000 + i], 8, 2, 128, dtype=BF16, device=cuda) for i in range(2)]
    alone = [_run(pal, c).clone() for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_run(pal, c))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, alone):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    # other lengths and queries, the same graph
    case, graph, out = cases[0], graphs[0], outs[0]
    case["lens"].copy_(torch.tensor([500, 50], dtype=torch.int32))
    case["lens_list"] = [500, 50]
    case["q"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert_chunk(out, case)


def test_append_then_attend(pal, cuda):
    """The operators as a step uses them: rotate and append the new tokens, then attend to the pages."""
    from rotary_reference import rotate64

    new, hist, hq, hkv, d, tpp = [1, 40, 3], [130, 9, 0], 8, 2, 128, 16
    lens = [n + h for n, h in zip(new, hist)]
    case = make_chunk_case(26, new, lens, hq, hkv, d, dtype=BF16, device=cuda, poison=False)
    T = sum(new)
    qkv = torch.randn((T, hq + 2 * hkv, d), generator=torch.Generator().manual_seed(1)).to(BF16)
    pos = torch.cat([torch.arange(h, h + n) for n, h in zip(new, hist)])
    seq = torch.cat([torch.full((n,), s) for s, n in enumerate(new)])
    freq = (1e4 ** (-torch.arange(d // 2, dtype=torch.float64) / (d // 2))).float()
    dq = qkv.to(cuda)
    _, _, q = pal.fill_kv_pages_rotary(dq[:, hq:hq + hkv], dq[:, hq + hkv:], case["k_pool"], case["v_pool"], case["table"], pos.to(cuda),
                                       seq.to(cuda), inv_freq=freq.to(cuda), queries=dq[:, :hq])
    case["q"] = q
    out = _run(pal, case)
    assert_chunk(out, case)  # (the pools now hold the rotated keys)
    page = case["table"].cpu().long()[seq, pos // tpp]
    k = case["k_pool"].cpu()[page, :, :, pos % tpp].reshape(T, hkv, d).double()
    assert (k - rotate64(qkv[:, hq:hq + hkv], pos, freq)).abs().max() <= 2.0 ** -8 * 8  # half a step of values below 8


def test_refusals(pal, cuda):
    case = make_chunk_case(27, [2, 3], [40, 50], 8, 2, 64, dtype=BF16, device=cuda)
    q, k, v, t, l, cu = (case[n] for n in ("q", "k_pool", "v_pool", "table", "lens", "cu"))
    call = pal.paged_attention_chunk
    for args, kw in [
        ((q[:, :7], k, v, t, l, cu), {}),
        ((q[..., :32], k, v, t, l, cu), {}),
        ((q.half(), k, v, t, l, cu), {}),
        ((q.float(), k.float(), v.float(), t, l, cu), {}),
        ((q[0], k, v, t, l, cu), {}),
        ((q, k[:1], v, t, l, cu), {}),
        ((q, k, v.transpose(2, 3), t, l, cu), {}),
        ((q, k, v, t[0], l, cu), {}),
        ((q, k, v, t, l[:1], cu), {}),
        ((q, k, v, t, l, cu[:2]), {}),
        ((q, k, v, t, l), {}),  # five rows, two sequences
        ((q, k, v, t, l, cu), dict(window=0)),
        ((q, k, v, t, l, cu), dict(window=-3)),
        ((q, k, v, t, l, cu), dict(window=4, causal=False)),
        ((q, k, v, t, l, cu), dict(out_dtype=FP16)),
        ((q, k, v, t, l, cu), dict(out=torch.empty((5, 8, 32), dtype=BF16, device=cuda))),
        ((q, k, v, t, l, cu), dict(out=torch.empty((5, 8, 64), device=cuda))),
    ]:
        with pytest.raises(ValueError):
            call(*args, **kw)
    with pytest.raises(TypeError):
        call(q, k, v, t.float(), l, cu)
    with pytest.raises(RuntimeError, match="no CPU path"):
        call(q, k, v, t, l.cpu(), cu)
    odd = torch.zeros((3, 2, 48, 16), dtype=BF16, device=cuda)
    with pytest.raises(RuntimeError, match="no kernel"):
        call(q[..., :48].contiguous(), torch.zeros((3, 2, 6, 16, 8), dtype=BF16, device=cuda), odd, t, l, cu)


def _poison(case, s, token, value, keys=True, dims=slice(None)):
    """Put `value` into a token of sequence s."""
    tpp = case["v_pool"].shape[3]
    page, slot = int(case["table"][s, token // tpp]), token % tpp
    if keys:
        case["k_pool"][page, :, :, slot] = value
    case["v_pool"][page, :, dims, slot] = value


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("hq,hkv,d,tpp", [(8, 2, 128, 16), (2, 2, 64, 32), (4, 1, 256, 16), (3, 1, 80, 32)])
def test_values_a_row_does_not_see_do_not_reach_it(pal, cuda, dtype, value, hq, hkv, d, tpp):
    """A token that is not finite: the rows before it, and those whose window starts after it, are untouched."""
    new, lens = [300, 5, 40], [430, 900, 40]
    for window in (None, 150):
        case = make_chunk_case(31, new, lens, hq, hkv, d, tpp=tpp, dtype=dtype, device=cuda, window=window)
        clean = _run(pal, case).clone()
        # (sequence, token, only values or keys too, which elements)
        spots = [(0, 130 + 77, False, slice(3, 4)), (0, 429, True, slice(None)), (1, 898, False, slice(None)), (2, 17, False, slice(0, 1))]
        if window:
            spots.append((0, 130 - 100, False, slice(5, 7)))  # seen by the first rows, then left behind
        for s, token, keys, dims in spots:
            _poison(case, s, token, value, keys, dims)
        out = _run(pal, case)
        row0 = 0
        for s, (n, L) in enumerate(zip(new, lens)):
            pos = torch.arange(L - n, L, device=cuda)
            sees = torch.zeros(n, dtype=torch.bool, device=cuda)
            for s2, token, _, _ in spots:
                if s2 == s:
                    sees |= (pos >= token) & ((pos - token < window) if window else True)
            rows, before = out[row0:row0 + n], clean[row0:row0 + n]
            # the same arithmetic on what they see: bit for bit
            assert torch.equal(rows[~sees].view(torch.int16), before[~sees].view(torch.int16)), (window, s)
            if bool(sees.any()):
                assert not torch.isfinite(rows[sees].float()).all(-1).any(), (window, s)
            row0 += n
        assert 0 < int((~torch.isfinite(out.float()).all(-1)).any(-1).sum()) < sum(new)


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, None), (FP16, None), (BF16, torch.float32), (FP16, torch.float32)])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("hq,hkv,d,tpp", [(8, 2, 128, 16), (2, 2, 64, 32), (4, 1, 256, 16), (3, 1, 80, 32)])
def test_values_that_are_not_finite_stay_in_their_elements(pal, cuda, dtype, out_dtype, value, hq, hkv, d, tpp):
    """An element of a value that is not finite makes that element of the rows that see it not finite and leaves all others bit for
    bit as they were, wherever the key lies: seen by all rows of an item, by some, in a part that is merged."""
    new, lens = [300, 5, 40, 1, 2], [430, 900, 40, 20000, 7]
    kw = dict(out_dtype=out_dtype)
    for window in (None, 150):
        case = make_chunk_case(35, new, lens, hq, hkv, d, tpp=tpp, dtype=dtype, device=cuda, window=window)
        clean = _run(pal, case, **kw).clone()
        # (sequence, token, kv head, element)
        spots = [(0, 200, 0, 3), (0, 429, hkv - 1, d - 1), (0, 131, 0, 17), (0, 257, hkv - 1, 17), (1, 898, 0, 8), (2, 17, 0, 0), (4, 6, 0, 31)]
        spots += [(0, 30, 0, 5), (0, 60, hkv - 1, 9)] if window else [(0, 2, 0, 5), (1, 100, 0, 20), (3, 12345, hkv - 1, 21), (3, 7, 0, 22)]
        hit = torch.zeros(clean.shape, dtype=torch.bool, device=cuda)
        for s, token, head, element in spots:
            page = int(case["table"][s, token // tpp])
            case["v_pool"][page, head, element, token % tpp] = value
            pos = torch.arange(lens[s] - new[s], lens[s], device=cuda)
            sees = (pos >= token) & ((pos - token < window) if window else True)
            rows = hit[sum(new[:s]):sum(new[:s + 1]), head * (hq // hkv):(head + 1) * (hq // hkv), element]
            rows |= sees[:, None]
        assert hit.any()
        for _ in range(2):
            out = _run(pal, case, **kw)
            assert not torch.isfinite(out[hit]).any()
            assert torch.equal(out[~hit], clean[~hit])
            if value != value:
                assert torch.isnan(out[hit]).all()


def test_infinities_of_both_signs_meet(pal, cuda):
    """In fp16 (no second product whose weights may be zero) an infinity that some rows of the item see stays one, and two of
    opposite signs make a NaN."""
    case = make_chunk_case(36, [100], [100], 4, 1, 64, dtype=FP16, device=cuda)
    for token, element, value in ((10, 3, float("inf")), (70, 3, -float("inf")), (40, 5, -float("inf"))):
        case["v_pool"][int(case["table"][0, token // 16]), 0, element, token % 16] = value
    out = _run(pal, case).float()
    assert torch.isfinite(out[:10]).all()
    assert (out[10:70, :, 3] == float("inf")).all() and torch.isnan(out[70:, :, 3]).all() and (out[40:, :, 5] == -float("inf")).all()
    assert torch.isfinite(out[..., 6:]).all()


@pytest.mark.parametrize("d,tpp", [(64, 16), (128, 32), (256, 16)])
@pytest.mark.parametrize("length", [1, 33, 129, 300])
def test_keys_that_are_not_numbers(pal, cuda, d, tpp, length):
    """A row that sees a NaN key is NaN, be it the only key, the only one of its tile or of a part of the tile, or one of many."""
    for new in (1, 40):
        if new > length:
            continue
        for first in {0, length // 2, length - 1}:
            case = make_chunk_case(33, [new], [length], 8, 2, d, tpp=tpp, dtype=BF16, device=cuda)
            clean = _run(pal, case).clone()
            for token in range(first, length):
                _poison(case, 0, token, float("nan"))
            out = _run(pal, case)
            sees = torch.arange(length - new, length, device=cuda) >= first
            assert torch.isnan(out[sees]).all() and torch.equal(out[~sees], clean[~sees])


def test_float32_output_with_a_value_that_is_not_finite(pal, cuda):
    case = make_chunk_case(32, [100], [400], 8, 2, 128, dtype=BF16, device=cuda)
    clean = _run(pal, case, out_dtype=torch.float32).clone()
    _poison(case, 0, 350, float("inf"))
    out = _run(pal, case, out_dtype=torch.float32)
    assert torch.equal(out[:50], clean[:50]) and not torch.isfinite(out[50:]).all(-1).any()


def test_pages_beyond_32_bit_offsets(pal, cuda):
    """Pages whose elements lie past 2^32 bytes and 2^31 elements of the pools: append with rotation, then attend, as in a small pool."""
    hq, hkv, d, tpp, n = 8, 8, 128, 16, 40
    pages = 2 ** 31 // (hkv * d * tpp) + 64
    g = torch.Generator().manual_seed(41)
    rand = lambda *shape: torch.randn(shape, generator=g).to(BF16).to(cuda)
    keys, values, queries = rand(n, hkv, d), rand(n, hkv, d), rand(n, hq, d)
    inv_freq = (10000.0 ** -(torch.arange(d // 2, dtype=torch.float64) / (d // 2))).float().to(cuda)
    pos = torch.arange(n, dtype=torch.int32, device=cuda)
    seq = torch.zeros(n, dtype=torch.int32, device=cuda)
    lens = torch.tensor([n], dtype=torch.int32, device=cuda)
    outs = []
    for total, ids in ((4, [2, 0, 3]), (pages, [pages - 1, 5, pages - 40])):
        k = torch.zeros((total, hkv, d // 8, tpp, 8), dtype=BF16, device=cuda)
        v = torch.zeros((total, hkv, d, tpp), dtype=BF16, device=cuda)
        table = torch.tensor([ids], dtype=torch.int32, device=cuda)
        _, _, q = pal.fill_kv_pages_rotary(keys, values, k, v, table, pos, seq, inv_freq=inv_freq, queries=queries)
        outs.append((k[ids].clone(), v[ids].clone(), pal.paged_attention_chunk(q, k, v, table, lens)))
        del k, v
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert outs[0][2].abs().sum() > 0
