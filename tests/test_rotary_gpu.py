"""rotary_embedding and fill_kv_pages_rotary against the rotation in 64 bits."""

import pytest
import torch

from rotary_reference import assert_rotated, rotate64

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _freqs(half, theta=5e5):
    return (theta ** (-torch.arange(half, dtype=torch.float64) / half)).float()


def _positions(tokens, sections, first, seed):
    g = torch.Generator().manual_seed(seed)
    axes = len(sections) if sections else 1
    pos = torch.randint(0, 3000, (axes, tokens), generator=g) + first
    return pos if axes > 1 else pos[0]


ROTATIONS = [
    # (tokens, heads, head_dim, rotary_dim, sections, order, pairing)
    (1, 1, 128, 128, None, "blocked", "half"),
    (1, 40, 128, 128, None, "blocked", "adjacent"),
    (7, 3, 64, 64, None, "blocked", "half"),
    (33, 5, 80, 80, [20, 20], "blocked", "half"),
    (33, 5, 80, 40, None, "blocked", "half"),           # half of 20: 8-byte vectors
    (33, 5, 80, 40, [8, 6, 6], "interleaved", "adjacent"),
    (65, 4, 128, 128, [16, 24, 24], "blocked", "half"),
    (65, 4, 128, 128, [24, 20, 20], "interleaved", "half"),
    (65, 4, 128, 64, [8, 8, 8, 8], "blocked", "adjacent"),
    (9, 2, 96, 96, [0, 48], "blocked", "half"),          # an axis without frequencies
    (130, 2, 256, 256, None, "blocked", "half"),
    (5, 2, 10, 6, None, "blocked", "half"),              # single elements, a row of no whole vector
    (5, 2, 7, 2, None, "blocked", "adjacent"),           # odd head
    (3, 2, 24, 8, None, "blocked", "half"),              # eight elements pass through in the last, half-empty unit
    (2000, 9, 128, 128, None, "blocked", "half"),        # several heads per thread
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,heads,head_dim,rotary_dim,sections,order,pairing", ROTATIONS)
def test_rotation(pal, cuda, tokens, heads, head_dim, rotary_dim, sections, order, pairing, dtype):
    g = torch.Generator().manual_seed(tokens * heads + head_dim)
    x = torch.randn((tokens, heads, head_dim), generator=g).to(dtype)
    freq, pos = _freqs(rotary_dim // 2), _positions(tokens, sections, 17, tokens)
    out = pal.rotary_embedding(x.to(cuda), pos.to(cuda), freq.to(cuda), sections=sections, section_order=order, pairing=pairing)
    assert out.is_contiguous() and out.dtype == dtype
    assert_rotated(out, x, pos, freq, sections, order, pairing)
    if rotary_dim < head_dim:
        assert torch.equal(out.cpu()[..., rotary_dim:], x[..., rotary_dim:])


@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("tokens,half,head_dim", [
    (2400, 367, 768), (2400, 368, 768), (2400, 369, 768), (2400, 375, 768), (2400, 376, 768), (2400, 384, 768),  # tables of 46 to 48 KB
    (2400, 512, 1024), (2367, 384, 768), (5, 4096, 8192), (300, 1001, 2003),
])
def test_wide_heads(pal, cuda, tokens, half, head_dim, pairing):
    """Heads up to the documented 8192 elements, whose angles fit a block's shared memory for sixteen tokens or for one."""
    x = torch.randn((tokens, 1, head_dim), generator=torch.Generator().manual_seed(half)).to(BF16)
    freq, pos = _freqs(half), _positions(tokens, None, 3, half)
    out = pal.rotary_embedding(x.to(cuda), pos.to(cuda), freq.to(cuda), pairing=pairing)
    assert_rotated(out, x, pos, freq, pairing=pairing)


@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64, torch.int16])
def test_far_and_negative_positions(pal, cuda, index_dtype):
    far = 30000 if index_dtype == torch.int16 else (2 ** 31 - 1 if index_dtype == torch.int32 else 2 ** 33 + 5)
    pos = torch.tensor([0, 1, -1, far, -far, far - 1], dtype=torch.int64)
    x = torch.randn((6, 2, 64), generator=torch.Generator().manual_seed(0)).to(FP16)
    freq = _freqs(32)
    out = pal.rotary_embedding(x.to(cuda), pos.to(index_dtype).to(cuda), freq.to(cuda), magnitude=1.25)
    assert_rotated(out, x, pos, freq, magnitude=1.25)


@pytest.mark.parametrize("kind", ["slice", "offset_one", "head_major", "broadcast_heads", "positions_strided"])
def test_strided_inputs(pal, cuda, kind):
    g = torch.Generator().manual_seed(3)
    T, H, D = 37, 4, 64
    pos, freq = _positions(T, [16, 8, 8], 5, 1), _freqs(32)
    dpos = pos.to(cuda)
    if kind == "slice":
        x = torch.randn((T, 3 * H, D), generator=g).to(BF16).to(cuda)[:, H:2 * H]
    elif kind == "offset_one":  # rows that start at odd elements: no vector access possible
        x = torch.randn((T * H * (D + 1) + 1,), generator=g).to(BF16).to(cuda)[1:].view(T, H, D + 1)[..., :D]
    elif kind == "head_major":
        x = torch.randn((H, T, D), generator=g).to(BF16).to(cuda).transpose(0, 1)
    elif kind == "broadcast_heads":
        x = torch.randn((T, 1, D), generator=g).to(BF16).to(cuda).expand(T, H, D)
    else:
        x = torch.randn((T, H, D), generator=g).to(BF16).to(cuda)
        dpos = torch.stack([pos, pos + 1], dim=-1).to(cuda)[..., 0]
    out = pal.rotary_embedding(x, dpos, freq.to(cuda), sections=[16, 8, 8])
    assert_rotated(out, x.cpu(), pos, freq, [16, 8, 8])


def test_in_place_and_strided_output(pal, cuda):
    T, H, D = 50, 6, 128
    x = torch.randn((T, H + 2, D), generator=torch.Generator().manual_seed(5)).to(BF16)
    pos, freq = _positions(T, None, 1000, 2), _freqs(64)
    buf = x.to(cuda)
    out = pal.rotary_embedding(buf[:, :H], pos.to(cuda), freq.to(cuda), out=buf[:, :H])
    assert out.data_ptr() == buf.data_ptr()
    assert_rotated(buf[:, :H], x[:, :H], pos, freq)
    assert torch.equal(buf[:, H:].cpu(), x[:, H:])  # the neighbours in the wider matrix stay


def test_negated_positions_undo_the_rotation_and_give_the_gradient(pal, cuda):
    T, H, D = 20, 3, 64
    g = torch.Generator().manual_seed(7)
    x = torch.randn((T, H, D), generator=g, dtype=torch.float64)
    grad = torch.randn((T, H, D), generator=g).to(FP16)
    pos, freq = _positions(T, None, 400, 3), _freqs(32)
    # the gradient's formula, and the same by differences of the definition: d(sum(grad * y)) / dx
    back = pal.rotary_embedding(grad.to(cuda), -pos.to(cuda), freq.to(cuda))
    assert_rotated(back, grad, -pos, freq)
    leaf = x.clone().requires_grad_(True)
    (rotate64_differentiable(leaf, pos, freq) * grad.double()).sum().backward()
    exact = rotate64(grad, -pos, freq)
    assert (leaf.grad - exact).abs().max() < 1e-12
    h = 1e-3
    for t, hh, d in [(0, 0, 0), (19, 2, 63), (7, 1, 31), (7, 1, 32)]:
        up, down = x.clone(), x.clone()
        up[t, hh, d] += h
        down[t, hh, d] -= h
        diff = ((rotate64(up, pos, freq) - rotate64(down, pos, freq)) * grad.double()).sum() / (2 * h)
        assert abs(diff - exact[t, hh, d]) < 1e-9  # the map is linear: only rounding separates the two


def rotate64_differentiable(x, pos, freq):
    half = freq.numel()
    angle = pos.double()[:, None] * freq.double()
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def test_nothing_to_rotate(pal, cuda):
    freq = _freqs(8).to(cuda)
    for shape in [(0, 4, 16), (3, 0, 16)]:
        x = torch.empty(shape, dtype=BF16, device=cuda)
        assert pal.rotary_embedding(x, torch.zeros(shape[0], dtype=torch.int32, device=cuda), freq).shape == shape


def test_rotation_refusals(pal, cuda):
    x = torch.zeros((4, 2, 16), dtype=BF16, device=cuda)
    pos, freq = torch.zeros(4, dtype=torch.int32, device=cuda), torch.ones(8, device=cuda)
    bad = [
        (dict(), dict(x=x[0])),
        (dict(), dict(x=x.float())),
        (dict(), dict(x=x.transpose(1, 2))),
        (dict(), dict(positions=pos[:3])),
        (dict(), dict(positions=pos[None].expand(2, 4))),
        (dict(), dict(inv_freq=torch.ones(9, device=cuda))),
        (dict(), dict(inv_freq=torch.ones(0, device=cuda))),
        (dict(), dict(inv_freq=freq.double())),
        (dict(sections=[4, 3]), dict(positions=pos[None].expand(2, 4))),
        (dict(sections=[9, -1]), dict(positions=pos[None].expand(2, 4))),
        (dict(sections=[2, 2, 2, 1, 1]), dict(positions=pos[None].expand(5, 4))),
        (dict(sections=[2, 6], section_order="interleaved"), dict(positions=pos[None].expand(2, 4))),
        (dict(sections=[4, 4]), dict()),
        (dict(section_order="other"), dict()),
        (dict(pairing="other"), dict()),
        (dict(out=torch.zeros((4, 2, 15), dtype=BF16, device=cuda)), dict()),
        (dict(out=torch.zeros((4, 2, 16), dtype=FP16, device=cuda)), dict()),
        (dict(out=torch.zeros((4, 1, 16), dtype=BF16, device=cuda).expand(4, 2, 16)), dict()),
    ]
    for options, changed in bad:
        args = dict(x=x, positions=pos, inv_freq=freq)
        args.update(changed)
        with pytest.raises(ValueError):
            pal.rotary_embedding(args["x"], args["positions"], args["inv_freq"], **options)
    with pytest.raises(TypeError):
        pal.rotary_embedding(x, pos.float(), freq)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pal.rotary_embedding(x.cpu(), pos, freq)
    with pytest.raises(RuntimeError, match="no CPU path"):
        pal.rotary_embedding(x, pos.cpu(), freq)


# ---------------------------------------------------------------------------------------------------------------------
# append with rotation
# ---------------------------------------------------------------------------------------------------------------------
def _batch(new, history, tpp, extra=3, seed=0):
    """(page table, pages in the pool, sequence of each token, position of each token)"""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-(n + h) // tpp) for n, h in zip(new, history)]
    perm = torch.randperm(sum(counts) + extra, generator=g).to(torch.int32)
    table = torch.full((len(new), max(counts) + 1), -1, dtype=torch.int32)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = perm[at:at + c]
        at += c
    seq = torch.cat([torch.full((n,), s) for s, n in enumerate(new)]).to(torch.int32)
    pos = torch.cat([torch.arange(h, h + n) for n, h in zip(new, history)]).to(torch.int32)
    return table, sum(counts) + extra, seq, pos


APPENDS = [
    # (new tokens, history, hq, hkv, head_dim, tokens_per_page)
    ([1], [0], 4, 1, 64, 16),
    ([1, 1, 1, 1, 1], [0, 15, 16, 300, 7], 8, 2, 128, 16),
    ([40, 1, 200], [3, 17, 8], 6, 2, 128, 16),
    ([64], [0], 2, 1, 128, 16),                   # octets up to the block border
    ([200], [5], 2, 2, 64, 32),                   # octets across it
    ([7, 8, 9, 15, 16, 17], [1, 0, 7, 9, 31, 32], 3, 3, 80, 16),
    ([71, 130], [0, 1], 4, 2, 96, 32),
    ([300], [60], 2, 2, 256, 16),
    ([33, 2], [1, 5], 2, 2, 32, 16),
    ([50], [3], 2, 2, 40, 8),                     # any head size and page size that fill_kv_pages takes
    ([50], [3], 2, 2, 64, 12),
    ([900, 3], [11, 0], 12, 4, 64, 16),
]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("slots", [False, True])
@pytest.mark.parametrize("new,history,hq,hkv,head_dim,tpp", APPENDS)
def test_append(pal, cuda, new, history, hq, hkv, head_dim, tpp, slots, dtype):
    table, pages, seq, pos = _batch(new, history, tpp, seed=sum(new))
    T = pos.numel()
    g = torch.Generator().manual_seed(T)
    qkv = torch.randn((T, hq + 2 * hkv, head_dim), generator=g).to(dtype)
    k_pool = torch.randn((pages, hkv, head_dim // 8, tpp, 8), generator=g).to(dtype)
    v_pool = torch.randn((pages, hkv, head_dim, tpp), generator=g).to(dtype)
    freq = _freqs(head_dim // 2)
    d = qkv.to(cuda)
    dk, dv = k_pool.to(cuda), v_pool.to(cuda)
    page = table[seq.long(), pos.long() // tpp].long()
    where = dict(slot_mapping=(page * tpp + pos.long() % tpp).to(cuda), positions=pos.to(cuda)) if slots else dict(
        page_table=table.to(cuda), current_token_write_positions=pos.to(cuda), query_to_seq_map=seq.to(cuda))
    q, k, v = d[:, :hq], d[:, hq:hq + hkv], d[:, hq + hkv:]
    rk, rv, rq = pal.fill_kv_pages_rotary(k, v, dk, dv, inv_freq=freq.to(cuda), queries=q, **where)
    assert rk is dk and rv is dv
    assert_rotated(rq, qkv[:, :hq], pos, freq)
    # the pools: exactly the new tokens' slots changed, values bit for bit
    slot = pos.long() % tpp
    expect_v = v_pool.clone()
    expect_v[page, :, :, slot] = qkv[:, hq + hkv:]
    assert torch.equal(dv.cpu().view(torch.int16), expect_v.view(torch.int16))
    got_k = dk.cpu()
    assert_rotated(got_k[page, :, :, slot].reshape(T, hkv, head_dim), qkv[:, hq:hq + hkv], pos, freq)
    got_k[page, :, :, slot] = k_pool[page, :, :, slot]
    assert torch.equal(got_k.view(torch.int16), k_pool.view(torch.int16))


def test_append_rotates_as_rotary_embedding_does(pal, cuda):
    """Every arrangement of the rotation, bit for bit, without queries, into a copy of the pools."""
    T, hkv, D, tpp = 77, 3, 128, 16
    table, pages, seq, pos = _batch([T], [9], tpp)
    g = torch.Generator().manual_seed(1)
    k = torch.randn((T, hkv, D), generator=g).to(BF16).to(cuda)
    v = torch.randn((T, hkv, D), generator=g).to(BF16).to(cuda)
    dk = torch.zeros((pages, hkv, D // 8, tpp, 8), dtype=BF16, device=cuda)
    dv = torch.zeros((pages, hkv, D, tpp), dtype=BF16, device=cuda)
    for options in (dict(), dict(pairing="adjacent"), dict(sections=[8, 12, 12], rotary=64), dict(sections=[24, 20, 20], section_order="interleaved"),
                    dict(magnitude=1.2), dict(rotary=40)):
        options = dict(options)
        freq = _freqs(options.pop("rotary", D) // 2).to(cuda)
        axes = len(options.get("sections", [0]))
        many = torch.stack([pos.to(cuda) + 5 * a for a in range(axes)])
        ak, av = pal.fill_kv_pages_rotary(k, v, dk, dv, table.to(cuda), pos.to(cuda), seq.to(cuda), inv_freq=freq, positions=many,
                                          inplace=False, **options)
        rotated = pal.rotary_embedding(k, many, freq, **options)
        fk, fv = pal.fill_kv_pages(rotated, v, dk.clone(), dv.clone(), table.to(cuda), pos.to(cuda), seq.to(cuda))
        assert torch.equal(ak.view(torch.int16), fk.view(torch.int16)) and torch.equal(av.view(torch.int16), fv.view(torch.int16))
        assert not dk.any() and not dv.any()


def test_tokens_without_a_destination_are_skipped(pal, cuda):
    T, hkv, D, tpp, pages = 40, 2, 64, 16, 4
    g = torch.Generator().manual_seed(2)
    q = torch.randn((T, 2, D), generator=g).to(FP16)
    k = torch.randn((T, hkv, D), generator=g).to(FP16)
    slots = torch.arange(T, dtype=torch.int64) + 3
    slots[[0, 7, 20]] = -1
    slots[[1, 30]] = pages * tpp
    freq, pos = _freqs(32), torch.arange(T)
    dk = torch.zeros((pages, hkv, D // 8, tpp, 8), dtype=FP16, device=cuda)
    dv = torch.zeros((pages, hkv, D, tpp), dtype=FP16, device=cuda)
    _, _, rq = pal.fill_kv_pages_rotary(k.to(cuda), k.to(cuda), dk, dv, slots.to(cuda), inv_freq=freq.to(cuda), positions=pos.to(cuda),
                                        queries=q.to(cuda))
    assert_rotated(rq, q, pos, freq)
    keep = ((slots >= 0) & (slots < pages * tpp)).nonzero().flatten()
    page, slot = slots[keep] // tpp, slots[keep] % tpp
    expect = torch.zeros((pages, hkv, D, tpp), dtype=FP16)
    expect[page, :, :, slot] = k[keep]
    assert torch.equal(dv.cpu(), expect)
    assert_rotated(dk.cpu()[page, :, :, slot].reshape(-1, hkv, D), k[keep], pos[keep], freq)
    # page-table form: a sequence index, a logical page and a page id out of range
    table = torch.tensor([[0, 99], [1, -1]], dtype=torch.int32)
    wp = torch.tensor([0, 16, 40, 5, 17, -3], dtype=torch.int32)
    sm = torch.tensor([0, 0, 0, 7, 1, 1], dtype=torch.int32)
    dk.zero_()
    dv.zero_()
    pal.fill_kv_pages_rotary(k[:6].to(cuda), k[:6].to(cuda), dk, dv, table.to(cuda), wp.to(cuda), sm.to(cuda), inv_freq=freq.to(cuda))
    expect = torch.zeros((pages, hkv, D, tpp), dtype=FP16)
    expect[0, :, :, 0] = k[0]
    assert torch.equal(dv.cpu(), expect)


@pytest.mark.parametrize("named_stream", [False, True])
@pytest.mark.parametrize("index_dtype", [torch.int32, torch.int64])
def test_slots_come_before_other_addresses(pal, cuda, index_dtype, named_stream):
    """Slots [sequences, tokens] beside write positions, a sequence map and a page table that say something else: the slots count."""
    B, L, hkv, D, tpp, pages = 4, 6, 2, 64, 16, 32
    g = torch.Generator().manual_seed(8)
    k, v = (torch.randn((B * L, hkv, D), generator=g).to(BF16).to(cuda) for _ in range(2))
    slots = torch.randperm(pages * tpp, generator=g)[:B * L].reshape(B, L)
    pos = torch.arange(L, dtype=torch.int32).repeat(B).to(cuda)
    seq = torch.arange(B, dtype=torch.int32).repeat_interleave(L).to(cuda)
    freq = _freqs(32).to(cuda)
    pools = lambda: (torch.zeros((pages, hkv, D // 8, tpp, 8), dtype=BF16, device=cuda), torch.zeros((pages, hkv, D, tpp), dtype=BF16, device=cuda))
    expect = pal.fill_kv_pages_rotary(k, v, *pools(), slots.flatten().to(torch.int64).to(cuda), inv_freq=freq, positions=pos)
    kw = dict(stream=torch.cuda.current_stream()) if named_stream else {}
    table = torch.arange(B, dtype=torch.int32, device=cuda)[:, None]
    for page_table in (None, table):
        got = pal.fill_kv_pages_rotary(k, v, *pools(), page_table, pos, seq, slot_mapping=slots.to(index_dtype).to(cuda), inv_freq=freq, positions=pos, **kw)
        for a, b in zip(got, expect):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_queries_in_place_of_a_fused_projection(pal, cuda):
    T, hq, hkv, D, tpp = 90, 4, 2, 128, 16
    table, pages, seq, pos = _batch([T], [2], tpp)
    x = torch.randn((T, hq + 2 * hkv, D), generator=torch.Generator().manual_seed(4)).to(BF16)
    buf = x.to(cuda)
    dk = torch.zeros((pages, hkv, D // 8, tpp, 8), dtype=BF16, device=cuda)
    dv = torch.zeros((pages, hkv, D, tpp), dtype=BF16, device=cuda)
    q = buf[:, :hq]
    pal.fill_kv_pages_rotary(buf[:, hq:hq + hkv], buf[:, hq + hkv:], dk, dv, table.to(cuda), pos.to(cuda), seq.to(cuda),
                             inv_freq=_freqs(64).to(cuda), queries=q, queries_out=q)
    assert_rotated(buf[:, :hq], x[:, :hq], pos, _freqs(64))
    assert torch.equal(buf[:, hq:].cpu(), x[:, hq:])


def test_append_refusals(pal, cuda):
    k = torch.zeros((4, 2, 64), dtype=BF16, device=cuda)
    dk = torch.zeros((3, 2, 8, 16, 8), dtype=BF16, device=cuda)
    dv = torch.zeros((3, 2, 64, 16), dtype=BF16, device=cuda)
    slots, pos, freq = torch.arange(4, device=cuda), torch.arange(4, device=cuda), torch.ones(32, device=cuda)
    call = lambda *a, **kw: pal.fill_kv_pages_rotary(*a, **{**dict(inv_freq=freq, positions=pos), **kw})
    for args, kw in [
        ((k, k, dk, dv, slots[:3]), {}),
        ((k, k, dk, dv, slots), dict(positions=None)),
        ((k, k, dk, dv), {}),
        ((k, k[:, :1], dk, dv, slots), {}),
        ((k.half(), k, dk, dv, slots), {}),
        ((k, k, dk, dv[:, :, :32], slots), {}),
        ((k, k, dk[:2], dv, slots), {}),
        ((k, k, dk, dv.transpose(2, 3).contiguous().transpose(2, 3), slots), {}),
        ((k, k, dk, dv, slots), dict(queries=k[:3])),
        ((k, k, dk, dv, slots), dict(queries=k[..., :32])),
        ((k, k, dk, dv, slots), dict(queries_out=k)),
        ((k.transpose(1, 2), k, dk, dv, slots), {}),
    ]:
        with pytest.raises(ValueError):
            call(*args, **kw)
    with pytest.raises(TypeError):
        call(k, k, dk, dv, slots.float())
    with pytest.raises(RuntimeError, match="no CPU path"):
        call(k, k, dk, dv, slots.cpu())
    assert not dk.any() and not dv.any()


def test_rotary_side_stream_and_graph(pal, cuda):
    """Captured and replayed with other inputs, and on a named stream with inputs that need a conversion."""
    T, hq, hkv, D, tpp = 24, 4, 2, 64, 16
    table, pages, seq, pos = _batch([T], [0], tpp)
    g = torch.Generator().manual_seed(6)
    x = torch.randn((T, hq + 2 * hkv, D), generator=g).to(BF16)
    buf, dpos, freq = x.to(cuda), pos.to(cuda), _freqs(32).to(cuda)
    dk = torch.zeros((pages, hkv, D // 8, tpp, 8), dtype=BF16, device=cuda)
    dv = torch.zeros((pages, hkv, D, tpp), dtype=BF16, device=cuda)
    dt, ds = table.to(cuda), seq.to(cuda)
    step = lambda **kw: pal.fill_kv_pages_rotary(buf[:, hq:hq + hkv], buf[:, hq + hkv:], dk, dv, dt, dpos, ds, inv_freq=freq,
                                                 queries=buf[:, :hq], **kw)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()[2]
    y = torch.randn(x.shape, generator=g).to(BF16)
    buf.copy_(y)
    dpos.copy_(torch.arange(8, 8 + T, dtype=torch.int32))
    dk.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert_rotated(out, y[:, :hq], torch.arange(8, 8 + T), _freqs(32))
    replayed = dk.clone()
    dk.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    dpos, ds = dpos.to(torch.int64), ds.to(torch.int64)
    step(stream=side)
    side.synchronize()
    assert torch.equal(dk.view(torch.int16), replayed.view(torch.int16))
