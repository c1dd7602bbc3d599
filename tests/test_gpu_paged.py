"""Paged append and paged attention against 64-bit restatements.

Tolerances follow from the arithmetic: u = 2^-8 (bf16) or 2^-11 (fp16) is the
relative error of one rounding. An append rounds once; its 32-bit rotation is
off by at most a few 2^-23 of |a| + |b|. An attention output is rounded once
(u |o|) and its weights may be rounded once to the cache's type (u sum p |v|).
The log-sum-exp carries the 32-bit sums of head_dim products and of the weights.
"""

import pytest
import torch

from oracle import paged as oracle

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _randn(gen, *shape, dtype=BF16):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _table(counts, width, pages, seed):
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    rows = []
    for c in counts:
        rows.append(order[:c] + [-1] * (width - c))
        order = order[c:]
    return torch.tensor(rows, dtype=torch.int32, device="cuda")


@pytest.fixture
def error_word(cuda):
    from layer_streaming import _native

    word = torch.zeros(1, dtype=torch.int32, device=cuda)
    _native.check(_native.lib().cb_set_error_word(word.data_ptr()), "cb_set_error_word")
    yield word
    torch.cuda.synchronize()
    _native.lib().cb_set_error_word(None)


@pytest.fixture
def workspace(cuda):
    from layer_streaming import ops

    return torch.zeros(ops.paged_attention_workspace_bytes(), dtype=torch.uint8, device=cuda)


# ------------------------------------------------------------------ attention
def _attention_case(lengths, hq, hk, d, page, dtype, seed=0, spread=1.0, garbage=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    counts = [-(-x // page) for x in lengths]
    pages, width = sum(counts) + 2, max(1, max(counts)) + 1
    table = _table(counts, width, pages, seed)
    k, v = _randn(gen, pages, hk, page, d, dtype=dtype), _randn(gen, pages, hk, page, d, dtype=dtype)
    if garbage is not None:  # everything that no length covers
        live = torch.zeros((pages, page), dtype=torch.bool)
        host = table.cpu()
        for b, length in enumerate(lengths):
            for j in range(length):
                live[host[b, j // page], j % page] = True
        dead = ~live.cuda()[:, None, :, None]
        k.masked_fill_(dead, garbage)
        v.masked_fill_(dead, garbage)
    q = (spread * torch.randn((len(lengths), hq, d), generator=gen, device="cuda")).to(dtype)
    return q, k, v, table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


def _run_attention(q, k, v, table, lengths, workspace, scale=None):
    from layer_streaming import ops

    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    lse = torch.full(q.shape[:2], float("nan"), device="cuda")
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    ops.paged_attention(q, k, v, table, lengths, scale, out, lse, workspace)
    return out, lse


def _check_attention(q, k, v, table, lengths, workspace, scale=None):
    out, lse = _run_attention(q, k, v, table, lengths, workspace, scale)
    torch.cuda.synchronize()
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, want_lse, weight, size = oracle.attention(q.cpu(), k.cpu(), v.cpu(), table.cpu(), lengths.cpu(), scale)
    u = oracle.UNIT[q.dtype]
    off = (out.cpu().double() - want).abs()
    assert (off <= 2.05 * u * weight + 1e-6).all(), float((off - 2.05 * u * weight).max())
    got = lse.cpu().double()
    empty = want_lse == -float("inf")
    assert torch.equal(got == -float("inf"), empty)
    tol = 2.0 ** -23 * (q.shape[-1] * size + lengths.cpu().double()[:, None] + 16)
    assert ((got - want_lse).abs()[~empty] <= tol[~empty]).all()
    assert int(torch.count_nonzero(workspace[:4096])) == 0  # the tickets
    return out, lse


LENGTHS = [1, 2, 15, 16, 17, 63, 64, 65, 0, 127, 128, 129, 500]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hk", [(8, 8), (8, 2), (6, 2), (7, 1), (8, 1), (12, 1), (16, 1), (40, 2)])
def test_attention_heads_and_types(workspace, dtype, d, hq, hk):
    _check_attention(*_attention_case(LENGTHS, hq, hk, d, 16, dtype), workspace)


@pytest.mark.parametrize("page", [1, 3, 8, 24, 48, 64, 100, 256, 1000])
def test_attention_page_sizes(workspace, page):
    _check_attention(*_attention_case([700, 1, 0, 333, page, page + 1], 8, 2, 128, page, BF16, seed=page), workspace)


@pytest.mark.parametrize("lengths", [[1], [0], [0, 0, 0], [5000], [3, 9000, 0, 64], [257] * 70])
def test_attention_batches(workspace, lengths):
    _check_attention(*_attention_case(lengths, 8, 2, 128, 32, BF16, seed=3), workspace)


def test_attention_many_sequences(workspace):
    lengths = [(37 * i) % 90 for i in range(1500)]  # more rows than threads of a CTA, every 90th empty
    _check_attention(*_attention_case(lengths, 2, 1, 64, 16, BF16, seed=4), workspace)


@pytest.mark.parametrize("garbage", [float("nan"), float("inf"), -float("inf")])
def test_attention_reads_nothing_behind_a_length(workspace, garbage):
    _check_attention(*_attention_case(LENGTHS, 8, 2, 128, 24, BF16, garbage=garbage), workspace)


def test_attention_peaked_scores(workspace):
    """Scores far apart (and all far below zero) keep the running maximum honest."""

    q, k, v, table, lengths = _attention_case([300, 1000, 77], 8, 2, 128, 16, BF16, spread=12.0)
    _check_attention(q, k, v, table, lengths, workspace)
    k.fill_(3.0)
    q.fill_(-3.0)
    _check_attention(q, k, v, table, lengths, workspace, scale=1.0)


def test_attention_strided_queries(workspace):
    q, k, v, table, lengths = _attention_case(LENGTHS, 8, 2, 128, 16, BF16)
    fused = torch.zeros((len(LENGTHS), 12, 128), dtype=BF16, device="cuda")
    fused[:, 2:10] = q
    got, lse = _run_attention(fused[:, 2:10], k, v, table, lengths, workspace)
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)  # head-major
    other, _ = _run_attention(turned, k, v, table, lengths, workspace)
    want, want_lse = _run_attention(q, k, v, table, lengths, workspace)
    assert torch.equal(got, want) and torch.equal(other, want) and torch.equal(lse, want_lse)


def test_attention_repeats_bit_for_bit_and_restores_its_workspace(workspace):
    case = _attention_case([4000, 3, 0, 900, 12], 8, 2, 128, 16, BF16)
    first = _run_attention(*case, workspace)
    _check_attention(*_attention_case(LENGTHS, 7, 1, 64, 24, FP16), workspace)
    for _ in range(3):
        again = _run_attention(*case, workspace)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_attention_without_lse(workspace):
    from layer_streaming import ops

    q, k, v, table, lengths = _attention_case(LENGTHS, 8, 2, 128, 16, BF16)
    out = torch.empty_like(q)
    torch.ops.cascade.paged_attention(q, k, v, table, lengths, 128 ** -0.5, out, None, workspace)
    assert torch.equal(out, _run_attention(q, k, v, table, lengths, workspace)[0])
    empty = q[:0]
    ops.paged_attention(empty, k, v, table[:0], lengths[:0], 1.0, empty.clone(), None, workspace)


def test_attention_offsets_beyond_32_bits(workspace):
    """A pool of more than 2^32 bytes and 2^31 elements; K and V share it."""

    pages, hk, page, d = 70000, 2, 128, 128
    pool = torch.empty((pages, hk, page, d), dtype=BF16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(5)
    held = [pages - 1, 3, pages - 2, 65537]
    for i in held:
        pool[i] = _randn(gen, hk, page, d)
    table = torch.tensor([held, [pages - 2, 65537, -1, -1]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([4 * page - 5, page + 9], dtype=torch.int32, device="cuda")
    q = _randn(gen, 2, 8, d)
    small = torch.tensor([[0, 1, 2, 3], [2, 3, -1, -1]], dtype=torch.int32, device="cuda")
    part = pool[torch.tensor(held, device="cuda")].contiguous()
    big, big_lse = _run_attention(q, pool, pool, table, lengths, workspace)
    want, want_lse = _check_attention(q, part, part, small, lengths, workspace)
    assert torch.equal(big, want) and torch.equal(big_lse, want_lse)


@pytest.mark.parametrize("d,group", [(64, 2), (128, 10)])
def test_attention_tables_of_two_to_the_31_positions(workspace, d, group):
    """Tables whose capacity passes 32-bit counts of places give what short ones give."""

    page, hk = 4096, 8
    q, k, v, table, lengths = _attention_case([5000, 1, 0, 9, 4097], group * hk, hk, d, page, BF16)
    wide = torch.full((5, 2 ** 31 // page - 1), -1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    want, want_lse = _check_attention(q, k, v, table, lengths, workspace)
    got, got_lse = _run_attention(q, k, v, wide, lengths, workspace)
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse)


def test_attention_reports_bad_tables_and_lengths(workspace, error_word):
    q, k, v, table, lengths = _attention_case([100, 60, 40], 8, 2, 128, 16, BF16)
    good, _ = _run_attention(q, k, v, table, lengths, workspace)
    assert int(error_word) == 0
    broken = table.clone()
    broken[1, 2] = k.shape[0]
    out, _ = _run_attention(q, k, v, broken, lengths, workspace)
    assert int(error_word) == 612
    assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    # the bad page's positions 32..47 are left out
    kept = torch.cat([broken[1, :2], broken[1, 3:4]]).view(1, -1)
    alone, _ = _check_attention(q[1:2], k, v, kept, torch.tensor([44], dtype=torch.int32, device="cuda"), workspace)
    torch.testing.assert_close(out[1].float(), alone[0].float(), rtol=2.0 ** -6, atol=2.0 ** -6)
    for wrong in (-5, table.shape[1] * 16 + 1):
        error_word.zero_()
        bad = lengths.clone()
        bad[0] = wrong
        out, _ = _run_attention(q, k, v, table.clamp(min=0), bad, workspace)
        assert int(error_word) == 611
        assert torch.equal(out[1], good[1]) and torch.equal(out[2], good[2])


def test_attention_refusals(workspace):
    from layer_streaming import ops

    q, k, v, table, lengths = _attention_case([5, 6], 8, 2, 128, 16, BF16)
    out, lse = torch.empty_like(q), torch.empty((2, 8), device="cuda")
    call = lambda **kw: ops.paged_attention(**{**dict(  # noqa: E731
        q=q, k_pages=k, v_pages=v, table=table, lengths=lengths, scale=1.0, out=out, lse=lse, workspace=workspace), **kw})
    call()
    for wrong in (
        {"q": q[:, :7], "out": out[:, :7].contiguous(), "lse": None},  # 7 heads over 2
        {"q": q[..., :64], "out": out[..., :64].contiguous()},
        {"table": table[:1]},
        {"lengths": lengths[:1]},
        {"out": out.transpose(0, 1).contiguous().transpose(0, 1)},
        {"workspace": workspace[:8]},
        {"q": q.float()},
        {"k_pages": k.to(FP16)},
        {"lengths": lengths.long()},
        {"table": table.long()},
        {"lse": lse[:1]},
        {"v_pages": v[:-1]},
        {"q": q.cpu()},
        {"q": q.transpose(1, 2).contiguous().transpose(1, 2)},
    ):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call(**wrong)
    wide = torch.zeros((2, 8, 32), dtype=BF16, device="cuda")
    pool = torch.zeros((4, 2, 16, 32), dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="head_dim=32"):
        call(q=wide, out=wide.clone(), k_pages=pool, v_pages=pool)


# --------------------------------------------------------------------- append
def _append_case(tokens, hq, hk, d, page, dtype, sequences=3, seed=0, longest=200):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    width = -(-longest // page)
    pages = sequences * width + 2
    table = _table([width] * sequences, width, pages, seed)
    # distinct (sequence, position) places
    places = torch.randperm(sequences * longest, generator=host)[:tokens]
    sequence, position = (places // longest).int().cuda(), (places % longest).int().cuda()
    fused = _randn(gen, tokens, hq + 2 * hk, d, dtype=dtype)
    k_pages, v_pages = _randn(gen, pages, hk, page, d, dtype=dtype), _randn(gen, pages, hk, page, d, dtype=dtype)
    return fused[:, :hq], fused[:, hq:hq + hk], fused[:, hq + hk:], sequence, position, table, k_pages, v_pages


def _freq(rotary, theta=10000.0):
    return (theta ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1))).float().cuda()


def _check_append(q, k, v, sequence, position, table, k_pages, v_pages, rotary, interleaved, factor=1.0):
    from layer_streaming import ops

    freq = _freq(rotary) if rotary else None
    q_out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    want_k, want_v = k_pages.cpu().clone(), v_pages.cpu().clone()
    ops.paged_append(q, k, v, freq, position, sequence, table, q_out, k_pages, v_pages, interleaved=interleaved,
                     factor=factor)
    torch.cuda.synchronize()
    host = lambda t: t.cpu()  # noqa: E731
    u, page = oracle.UNIT[q.dtype], k_pages.shape[2]

    def expected(x):
        x = host(x)
        return oracle.rotate(x, freq.cpu(), host(position), interleaved, factor) if rotary else x.double()

    size = lambda x: 2 * abs(factor) * host(x).double().abs().amax(-1, keepdim=True)  # noqa: E731
    live = host(position) >= 0
    for got, x in ((q_out.cpu(), q),):
        want = expected(x) * live[:, None, None]
        assert ((got.double() - want).abs() <= 1.01 * u * want.abs() + 2.0 ** -21 * size(x) + 1e-7).all()
    turned = expected(k)
    got_k, got_v = k_pages.cpu(), v_pages.cpu()
    for n in range(q.shape[0]):
        if not live[n]:
            continue
        j = int(position[n])
        at = int(table[int(sequence[n]) if sequence is not None else n, j // page])
        row = got_k[at, :, j % page].double()
        assert ((row - turned[n]).abs() <= 1.01 * u * turned[n].abs() + 2.0 ** -21 * size(k)[n] + 1e-7).all()
        want_k[at, :, j % page] = got_k[at, :, j % page]
        want_v[at, :, j % page] = v[n].cpu()
    assert torch.equal(got_k, want_k) and torch.equal(got_v, want_v)  # nothing else was touched
    return q_out


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rotary", [(128, 128), (128, 64), (128, 16), (64, 64), (96, 32), (256, 256), (128, 0)])
def test_append_rotations(cuda, dtype, interleaved, d, rotary):
    _check_append(*_append_case(37, 8, 2, d, 16, dtype), rotary, interleaved, factor=1.0 if rotary != 64 else 0.7)


@pytest.mark.parametrize("page", [1, 7, 24, 64, 300])
@pytest.mark.parametrize("tokens", [1, 5, 300])
def test_append_pages_and_tokens(cuda, page, tokens):
    _check_append(*_append_case(tokens, 4, 4, 64, page, BF16, seed=tokens), 64, False)


@pytest.mark.parametrize("hq,hk", [(1, 1), (7, 1), (40, 8), (3, 3)])
def test_append_heads(cuda, hq, hk):
    _check_append(*_append_case(19, hq, hk, 128, 16, BF16, seed=2), 128, False)


def test_append_far_positions(cuda):
    """The angle stays right where a 32-bit product would be off by 0.03 rad."""

    q, k, v, _, _, _, _, _ = _append_case(6, 4, 2, 64, 16, FP16)
    position = torch.tensor([0, 131071, 1048575, 262143, 999983, 524289], dtype=torch.int32, device="cuda")
    page = 1 << 16
    pool = lambda: torch.zeros((18, 2, page, 64), dtype=FP16, device="cuda")  # noqa: E731
    table = torch.arange(17, dtype=torch.int32, device="cuda").view(1, -1)
    sequence = torch.zeros(6, dtype=torch.int32, device="cuda")
    _check_append(q, k, v, sequence, position, table, pool(), pool(), 64, False)


def test_append_padding_and_default_sequence(cuda):
    q, k, v, _, position, table, k_pages, v_pages = _append_case(3, 8, 2, 128, 16, BF16)
    position = position.clone()
    position[1] = -1
    q_out = _check_append(q, k, v, None, position, table, k_pages, v_pages, 128, False)
    assert int(torch.count_nonzero(q_out[1])) == 0


def test_append_in_place_and_cache_only(cuda):
    from layer_streaming import ops

    q, k, v, sequence, position, table, k_pages, v_pages = _append_case(9, 8, 2, 128, 16, BF16)
    freq = _freq(128)
    out, pools = torch.empty(q.shape, dtype=BF16, device="cuda"), [k_pages.clone(), v_pages.clone()]
    torch.ops.cascade.paged_append(q, k, v, freq, position, sequence, table, out, k_pages, v_pages)
    same = q.contiguous()
    ops.paged_append(same, k, v, freq, position, sequence, table, same, *pools)
    assert torch.equal(same, out) and torch.equal(pools[0], k_pages) and torch.equal(pools[1], v_pages)
    # a contiguous cache [heads, positions, dim] seen as tokens: keys are taken as they are
    cache = _randn(torch.Generator(device="cuda").manual_seed(1), 2, 9, 128)
    ops.paged_append(None, cache.transpose(0, 1), cache.transpose(0, 1), None, position, sequence, table, None, *pools)
    for n in range(9):
        at, j = int(table[int(sequence[n]), int(position[n]) // 16]), int(position[n]) % 16
        assert torch.equal(pools[0][at, :, j], cache[:, n]) and torch.equal(pools[1][at, :, j], cache[:, n])


def test_append_reports_bad_places(cuda, error_word):
    from layer_streaming import ops

    for field, value in (("sequence", 3), ("sequence", -1), ("position", 13 * 16), ("table", -1), ("table", 10 ** 6)):
        q, k, v, sequence, position, table, k_pages, v_pages = _append_case(4, 8, 2, 128, 16, BF16)
        sequence, position, table = sequence.clone(), position.clone(), table.clone()
        if field == "table":
            table[int(sequence[2]), int(position[2]) // 16] = value
        else:
            {"sequence": sequence, "position": position}[field][2] = value
        before = k_pages.clone()
        ops.paged_append(q, k, v, _freq(128), position, sequence, table, torch.empty_like(q.contiguous()), k_pages, v_pages)
        assert int(error_word) == 601
        assert int((k_pages != before).any(-1).any(1).sum()) <= 3  # the others were written
        error_word.zero_()


def test_append_refusals(cuda):
    from layer_streaming import ops

    q, k, v, sequence, position, table, k_pages, v_pages = _append_case(4, 8, 2, 128, 16, BF16)
    args = dict(q=q, k=k, v=v, inv_freq=_freq(128), position=position, sequence=sequence, table=table,
                q_out=torch.empty_like(q.contiguous()), k_pages=k_pages, v_pages=v_pages)
    ops.paged_append(**args)
    for wrong in (
        {"q_out": None}, {"v": v[:, :1]}, {"k": k.float()}, {"q": q[..., :64]}, {"inv_freq": _freq(24)},
        {"inv_freq": _freq(256)}, {"position": position.long()}, {"position": position[:2]}, {"sequence": sequence[:3]},
        {"k_pages": k_pages[:, :1].contiguous()}, {"v_pages": v_pages[1:]}, {"sequence": None}, {"k": k.cpu()},
        {"q_out": q}, {"inv_freq": _freq(128).double()}, {"k_pages": k_pages.transpose(1, 2)},
    ):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.paged_append(**{**args, **wrong})


# ----------------------------------------------------------- both, in a graph
def test_append_then_attention_in_a_graph_on_a_side_stream(workspace):
    """A captured step: append at the counted position, attend, on another stream."""

    from layer_streaming import ops

    q, k, v, sequence, position, table, k_pages, v_pages = _append_case(3, 8, 2, 128, 16, BF16, longest=64)
    sequence = torch.arange(3, dtype=torch.int32, device="cuda")
    position = torch.tensor([4, 20, 33], dtype=torch.int32, device="cuda")
    lengths = position + 1
    q_out, out = torch.empty_like(q.contiguous()), torch.empty_like(q.contiguous())
    lse = torch.empty((3, 8), device="cuda")
    freq, scale = _freq(128), 128 ** -0.5

    def step():
        ops.paged_append(q, k, v, freq, position, sequence, table, q_out, k_pages, v_pages)
        ops.paged_attention(q_out, k_pages, v_pages, table, lengths, scale, out, lse, workspace)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
        for _ in range(3):
            position += 1
            lengths += 1
            graph.replay()
        side.synchronize()
    want, _, weight, _ = oracle.attention(q_out.cpu(), k_pages.cpu(), v_pages.cpu(), table.cpu(), lengths.cpu(), scale)
    assert ((out.cpu().double() - want).abs() <= 2.05 * 2.0 ** -8 * weight + 1e-6).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_at_any_int32_position(cuda, dtype, interleaved):
    """The largest angle is the position itself, which 32 bits hold to within 64 rad at 2^31."""

    position = [0, 1048577, 4194303, 7000001, 16777217, 123456789, 2 ** 30 + 1, 2 ** 31 - 2 ** 16 - 1]
    gen = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn((len(position), 4, 64), generator=gen, device="cuda").to(dtype)
    page = 1 << 16
    table = torch.full((1, 2 ** 31 // page - 1), -1, dtype=torch.int32)
    for n, j in enumerate(position):
        table[0, j // page] = n
    pool = lambda: torch.zeros((len(position), 1, page, 64), dtype=dtype, device="cuda")  # noqa: E731
    sequence = torch.zeros(len(position), dtype=torch.int32, device="cuda")
    _check_append(qkv[:, :2], qkv[:, 2:3], qkv[:, 3:], sequence, torch.tensor(position, dtype=torch.int32, device="cuda"),
                  table.cuda(), pool(), pool(), 64, interleaved)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("d,group", [(64, 3), (128, 8), (128, 16), (64, 16)])
def test_attention_weights_are_not_rounded_to_the_cache_type(workspace, dtype, d, group):
    """Outputs that nearly vanish: the bound leaves no room for weights of 8 or 11 bits."""

    case = oracle.cancelling_case(dtype, d, group, [16, 32, 48, 2], 24)
    want, _, weight, _ = oracle.attention(*case, 1.0)
    out, _ = _run_attention(*(x.cuda() for x in case), workspace, scale=1.0)
    assert ((out.cpu().double() - want).abs() <= oracle.cancelling_bound(dtype, want, weight, case[-1])).all()
