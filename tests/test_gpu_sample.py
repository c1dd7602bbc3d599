"""Sampling against the definition in 64 bits.

The 32-bit exponent argument is off by at most 2^-23 of its size (28 at most
where a weight counts) and expf by 2 ulp, so a weight's relative error, and with
it every share of the mass, stays below 28 * 2^-23 + 2^-21 < 5e-6: the slack
within which a threshold may fall on either side.
"""

import math

import pytest
import torch

from oracle import paged as oracle

pytestmark = pytest.mark.gpu

SLACK = 5e-6
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _f(values):
    return None if values is None else torch.tensor(values, dtype=torch.float32, device="cuda")


def _i(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device="cuda")


def _sample(logits, temperature=None, top_k=None, top_p=None, min_p=None, uniform=None):
    from layer_streaming import ops

    rows = logits.shape[0]
    uniform = [0.5] * rows if uniform is None else uniform
    tokens = torch.full((rows,), -7, dtype=torch.int64, device="cuda")
    logprobs = torch.full((rows,), float("nan"), device="cuda")
    ops.sample(logits, _f(temperature), _i(top_k), _f(top_p), _f(min_p), _f(uniform), tokens, logprobs)
    return tokens.tolist(), logprobs.tolist()


def _check(logits, temperature=None, top_k=None, top_p=None, min_p=None, uniform=None):
    rows = logits.shape[0]
    uniform = [0.5] * rows if uniform is None else uniform
    tokens, logprobs = _sample(logits, temperature, top_k, top_p, min_p, uniform)
    host = logits.cpu()
    pick = lambda v, r, default: default if v is None else float(torch.tensor(v[r], dtype=torch.float32))  # noqa: E731
    for r in range(rows):
        wrong = oracle.sample_check(host[r], pick(temperature, r, 1.0), 0 if top_k is None else top_k[r],
                                    pick(top_p, r, 1.0), pick(min_p, r, 0.0), pick(uniform, r, 0.5), tokens[r],
                                    logprobs[r], SLACK)
        assert wrong is None, (r, wrong)
    return tokens, logprobs


def _logits(rows, vocab, dtype, seed=0, std=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (std * torch.randn((rows, vocab), generator=gen, device="cuda")).to(dtype)


def _u(rows, seed=0):
    return torch.rand(rows, generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 4097, 32003, 128256])
def test_all_filters(cuda, dtype, vocab):
    rows = 12
    k = [0, 1, 2, 5, 50, 64, 100, 1000, vocab, vocab + 5, -3, 7]
    p = [1.0, 0.9, 0.5, 0.1, 0.99, 0.0, 1.5, 0.8, 0.95, 0.3, 0.9, 1.0]
    m = [0.0, 0.0, 0.05, 0.0, 0.01, 0.0, 0.3, 0.0, 1.0, 0.0, 2.0, -1.0]
    t = [1.0, 0.7, 1.3, 0.2, 5.0, 1.0, 0.0, 0.9, 1.0, 2.0, 1.0, -1.0]
    for seed in range(3):
        _check(_logits(rows, vocab, dtype, seed), t, k, p, m, _u(rows, seed))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("field", ["temperature", "top_k", "top_p", "min_p", None])
def test_one_filter_at_a_time(cuda, dtype, field):
    rows = 8
    value = {"temperature": [0.3, 0.5, 0.8, 1.0, 1.5, 3.0, 30.0, 0.0], "top_k": [1, 2, 3, 10, 40, 200, 5000, 0],
             "top_p": [0.01, 0.2, 0.5, 0.8, 0.9, 0.95, 0.999, 1.0], "min_p": [0.0, 1e-4, 1e-3, 0.01, 0.05, 0.2, 0.9, 1.0]}
    _check(_logits(rows, 50257, dtype, 9), uniform=_u(rows, 3), **({field: value[field]} if field else {}))


@pytest.mark.parametrize("vocab", [200000, 262144, 1000003])
def test_large_vocabularies(cuda, vocab):
    _check(_logits(3, vocab, torch.float32, 2), [1.0, 0.8, 1.2], [0, 40, 0], [1.0, 0.9, 0.95], None, _u(3, 8))


def test_greedy_ties_go_to_the_lowest_index(cuda):
    logits = torch.zeros((4, 5000), device="cuda")
    logits[0, [4999, 17, 900]] = 2.5
    logits[1, 4999] = 1.0
    logits[3, 0] = -0.0
    for u in (0.0, 0.999):
        tokens, logprobs = _sample(logits, temperature=[0.0, 0.0, 0.0, 0.0], uniform=[u] * 4)
        assert tokens == [17, 4999, 0, 0] and logprobs == [0.0] * 4
        assert _sample(logits, top_k=[1] * 4, uniform=[u] * 4)[0] == [17, 4999, 0, 0]


def test_equal_logits_are_cut_in_index_order(cuda):
    """All logits equal: every cut falls inside one tie group of the whole vocabulary."""

    vocab = 40000
    logits = torch.full((6, vocab), 1.25, device="cuda")
    k = [7, 1000, 0, 0, 39999, 3]
    p = [1.0, 1.0, 0.5, 0.0001, 1.0, 0.5]
    kept = [7, 1000, 20000, 5, 39999, 2]  # 0.0001 is 1678 / 2^24 in fixed point: 4.0006 tokens, rounded up
    for u in (0.0, 0.25, 0.5, 0.9999999):
        u32 = float(torch.tensor(u, dtype=torch.float32))
        tokens, logprobs = _sample(logits, top_k=k, top_p=p, uniform=[u] * 6)
        assert tokens == [int(u32 * 2 ** 24) * n // 2 ** 24 for n in kept]
        assert logprobs == pytest.approx([-math.log(n) for n in kept], abs=2e-6)


def test_few_distinct_values(cuda):
    """Large tie groups at several levels, scattered over the vocabulary."""

    gen = torch.Generator(device="cuda").manual_seed(4)
    for dtype in TYPES:
        logits = (torch.randint(0, 4, (6, 30011), generator=gen, device="cuda").float() * 0.75).to(dtype)
        _check(logits, [1.0, 0.5, 2.0, 1.0, 1.0, 1.0], [0, 9000, 20000, 0, 12345, 7500], [0.5, 0.9, 1.0, 0.2, 0.7, 1.0],
               [0.0, 0.0, 0.0, 0.3, 0.0, 0.9], _u(6, 1))


def test_masked_and_odd_logits(cuda):
    inf, nan = float("inf"), float("nan")
    vocab = 3001
    logits = _logits(9, vocab, torch.float32, 5)
    logits[0] = -inf
    logits[1] = nan
    logits[2, 1:] = -inf                                  # one choice
    logits[3, :] = -inf
    logits[3, [5, 2000]] = torch.tensor([1.0, 2.0], device="cuda")
    logits[4, 100] = inf
    logits[5, [100, 200]] = inf
    logits[6, ::2] = nan
    logits[7] = torch.finfo(torch.float32).min            # the type's lowest value everywhere
    logits[8, 3:] = torch.finfo(torch.float32).min
    u = _u(9, 7)
    tokens, logprobs = _sample(logits, top_p=[0.9] * 9, uniform=u)
    assert tokens[0] == tokens[1] == -1 and logprobs[0] == logprobs[1] == -inf
    assert tokens[2] == 0 and logprobs[2] == 0.0
    assert tokens[3] in (5, 2000)
    assert tokens[4] == 100 and logprobs[4] == 0.0
    assert tokens[5] in (100, 200) and logprobs[5] == pytest.approx(-math.log(2), abs=1e-6)
    assert tokens[6] % 2 == 1
    assert 0 <= tokens[7] < vocab and logprobs[7] == pytest.approx(-math.log(math.ceil(0.9 * vocab)), abs=1e-3)
    assert tokens[8] in (0, 1, 2)
    for dtype in TYPES:
        rows = torch.full((2, 500), torch.finfo(dtype).min, device="cuda", dtype=dtype)
        rows[0, 77] = 1.0
        tokens, _ = _sample(rows, uniform=[0.99, 0.0])
        assert tokens == [77, 0]


def test_odd_parameters(cuda):
    nan, inf = float("nan"), float("inf")
    logits = _logits(8, 700, torch.float32, 6)
    best = logits.argmax(1).tolist()
    tokens, _ = _sample(logits, temperature=[nan, inf, 1e-42, 1.0, 1.0, 1.0, 1.0, 1.0], top_k=[0] * 8,
                        top_p=[1.0, 1.0, 1.0, nan, -1.0, 1.0, 1.0, 1.0], min_p=[0.0, 0.0, 0.0, 0.0, 0.0, nan, inf, 0.0],
                        uniform=[0.3, 0.5, 0.7, 0.2, 0.9, 0.1, 0.4, nan])
    assert tokens[0] == best[0] and tokens[2] == best[2] and tokens[4] == best[4] and tokens[6] == best[6]
    assert tokens[1] == 350  # flat over the vocabulary
    assert all(0 <= t < 700 for t in tokens)
    low, _ = _sample(logits, uniform=[-1.0] * 8)
    high, _ = _sample(logits, uniform=[1.0] * 8)
    assert low == _sample(logits, uniform=[0.0] * 8)[0]
    assert high == _sample(logits, uniform=[1.0 - 2.0 ** -24] * 8)[0]


def test_frequencies(cuda):
    """4096 evenly spaced uniforms draw each token in proportion to its probability."""

    n = 4096
    row = torch.tensor([0.5, -1.0, 2.0, 1.5, -3.0], device="cuda")
    logits = row.repeat(n, 1)
    tokens, _ = _sample(logits, temperature=[1.7] * n, uniform=[(i + 0.5) / n for i in range(n)])
    share = torch.bincount(torch.tensor(tokens), minlength=5).double() / n
    want = torch.softmax(row.cpu().double() / 1.7, 0)
    assert ((share - want).abs() <= 1.0 / n + 1e-6).all()
    assert tokens == sorted(tokens)  # index order


def test_strided_rows_and_optional_outputs(cuda):
    from layer_streaming import ops

    wide = _logits(10, 9000, torch.bfloat16, 8)
    view = wide[::2, 11:8011]  # rows start on odd addresses
    u = _u(5, 2)
    want = _check(view.contiguous(), top_p=[0.9] * 5, uniform=u)
    assert _sample(view, top_p=[0.9] * 5, uniform=u) == want
    tokens = torch.empty(5, dtype=torch.int64, device="cuda")
    torch.ops.cascade.sample(view, None, None, _f([0.9] * 5), None, _f(u), tokens, None)
    assert tokens.tolist() == want[0]
    ops.sample(view[:0], None, None, None, None, _f([]), tokens[:0], None)


def test_repeats_bit_for_bit(cuda):
    logits = _logits(64, 128256, torch.bfloat16, 12, std=2.0)
    first = _sample(logits, top_p=[0.95] * 64, uniform=_u(64, 5))
    for _ in range(3):
        assert _sample(logits, top_p=[0.95] * 64, uniform=_u(64, 5)) == first


@pytest.mark.parametrize("rows,vocab,dtype", [(700, 9000, torch.float32), (90, 128256, torch.bfloat16)])
def test_a_large_mixed_batch_equals_its_rows_one_at_a_time(cuda, rows, vocab, dtype):
    """Large batches are ordered by cost and share CTAs; the answers are the rows' own."""

    logits = _logits(rows, vocab, dtype, 3)
    host = torch.Generator().manual_seed(1)
    pick = lambda values: [values[i] for i in torch.randint(0, len(values), (rows,), generator=host).tolist()]  # noqa: E731
    t, k = pick([0.0, 0.7, 1.0, 1.6]), pick([0, 0, 1, 40, 300, 900])
    p, m, u = pick([1.0, 0.9, 0.5]), pick([0.0, 0.0, 0.05]), _u(rows, 4)
    together = _sample(logits, t, k, p, m, u)
    for r in range(0, rows, 7):
        one = _sample(logits[r:r + 1], t[r:r + 1], k[r:r + 1], p[r:r + 1], m[r:r + 1], u[r:r + 1])
        assert one[0][0] == together[0][r] and one[1][0] == together[1][r]
    _check(logits[:16], t[:16], k[:16], p[:16], m[:16], u[:16])
    # all rows of one kind
    for kinds in ({"temperature": [0.0] * rows}, {"top_k": [5] * rows}, {"top_p": [0.3] * rows}, {}):
        whole, some = _sample(logits, uniform=u, **kinds), _sample(logits[:3], uniform=u[:3], **{
            key: value[:3] for key, value in kinds.items()})
        assert whole[0][:3] == some[0] and whole[1][:3] == some[1] and -7 not in whole[0]


def test_refusals(cuda):
    from layer_streaming import ops

    logits = _logits(4, 100, torch.float32)
    tokens = torch.empty(4, dtype=torch.int64, device="cuda")
    args = dict(logits=logits, temperature=None, top_k=None, top_p=None, min_p=None, uniform=_f([0.5] * 4),
                tokens=tokens, logprobs=None)
    ops.sample(**args)
    with pytest.raises(RuntimeError, match="vocab"):
        ops.sample(**{**args, "logits": torch.zeros((1, 2080001), device="cuda").expand(4, -1)})
    for wrong in ({"logits": logits[0]}, {"logits": logits.double()}, {"logits": logits.t()}, {"logits": logits.cpu()},
                  {"uniform": _f([0.5] * 3)}, {"tokens": tokens.int()}, {"top_k": torch.zeros(4, dtype=torch.int64, device="cuda")},
                  {"temperature": _f([1.0])}, {"logprobs": torch.empty(4, dtype=torch.float64, device="cuda")},
                  {"top_p": torch.ones(4)}):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.sample(**{**args, **wrong})


@pytest.mark.parametrize("vocab", [5000, 50257, 262144])
@pytest.mark.parametrize("levels", [3, 64, 1000])
def test_top_p_where_many_tokens_share_a_logit(cuda, vocab, levels):
    """Few distinct logits: whole levels fill the boundary's interval and its lists."""

    gen = torch.Generator(device="cuda").manual_seed(levels)
    step = torch.randint(0, levels, (7, vocab), generator=gen, device="cuda")
    p = [0.001, 0.3, 0.5, 0.9, 0.99, 0.9999, 0.7]
    m = [0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.2]
    _check(step * (6.0 / levels), [1.0, 0.5, 2.0, 1.0, 1.0, 0.3, 1.0], None, p, m, _u(7, levels))


@pytest.mark.parametrize("width", [1e-6, 1e-3, 0.3, 8.0, 24.0])
def test_top_p_over_crowded_and_wide_logits(cuda, width):
    """From logits a few ulp apart to some where only the largest have weight."""

    gen = torch.Generator(device="cuda").manual_seed(4)
    logits = 1.0 + width * torch.rand((6, 100000), generator=gen, device="cuda")
    p = [0.01, 0.4, 0.8, 0.95, 0.999, 0.99999]
    _check(logits, [1.0, 1.0, 0.6, 1.5, 1.0, 1.0], None, p, None, _u(6, 1))


@pytest.mark.parametrize("dtype", TYPES)
def test_top_p_reads_nothing_into_invalid_logits(cuda, dtype):
    """A vocabulary whose halves are NaN and -inf samples as the finite rest does."""

    logits = _logits(4, 3 * 20011, dtype, 6, std=2.0)
    full = logits.clone()
    full[:, 1::3] = float("nan")
    full[:, 2::3] = -float("inf")
    rest = logits[:, 0::3].contiguous()
    p, u = [0.3, 0.9, 0.99, 0.9999], _u(4, 6)
    got, got_lp = _sample(full, None, None, p, None, u)
    want, want_lp = _check(rest, None, None, p, None, u)
    assert got == [3 * w for w in want] and got_lp == want_lp


def test_top_p_in_large_batches(cuda):
    """Rows of every kind in an order of their cost, some with more kept tokens than lists hold."""

    rows, vocab = 320, 32003
    logits = _logits(rows, vocab, torch.bfloat16, 8, std=2.0)
    t = [0.0 if r % 7 == 0 else 0.4 + 0.2 * (r % 9) for r in range(rows)]
    k = [40 if r % 5 == 0 else 0 for r in range(rows)]
    p = [1.0 if r % 3 == 0 else 0.5 + 0.49 * (r % 11) / 10 for r in range(rows)]
    m = [0.05 if r % 4 == 0 else 0.0 for r in range(rows)]
    _check(logits, t, k, p, m, _u(rows, 8))


@pytest.mark.parametrize("vocab", [9, 40, 700, 8000])
@pytest.mark.parametrize("infinite", [False, True])
def test_rows_of_one_cta_agree_on_their_largest_logit(cuda, vocab, infinite):
    """Without a filter, and with an infinite logit, a row goes from its largest logit straight to the
    sums, which use the same shared words; in a short row most warps have no logits and arrive early.
    The other logits lie 60 below the largest (e^-60 has no weight), so the answer is known."""

    from layer_streaming import ops

    rows = 2000
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    best = torch.randint(0, vocab, (rows, 1), generator=gen, device="cuda")
    logits = torch.rand((rows, vocab), generator=gen, device="cuda") - 62.0
    logits.scatter_(1, best, float("inf") if infinite else 0.0)
    uniform = torch.rand(rows, generator=gen, device="cuda")
    tokens, logprobs = torch.empty(rows, dtype=torch.int64, device="cuda"), torch.empty(rows, device="cuda")
    for _ in range(30):
        tokens.fill_(-7)
        ops.sample(logits, None, None, None, None, uniform, tokens, logprobs)
        assert torch.equal(tokens, best[:, 0]) and int(torch.count_nonzero(logprobs)) == 0
