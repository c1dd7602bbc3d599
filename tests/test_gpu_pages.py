"""Page bookkeeping on the device against the same steps on Python lists:
every table entry, length, count and page content is equal."""

import random

import pytest
import torch

from oracle.paged import Pages

pytestmark = pytest.mark.gpu

LAYERS, HEADS, DIM = 2, 2, 16


class Device:
    """The device state of an oracle state; page p of every block is filled with its content's number."""

    def __init__(self, oracle, dtype=torch.bfloat16):
        from layer_streaming import ops

        as_int = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        self.table, self.lengths, self.ref = as_int(oracle.table), as_int(oracle.lengths), as_int(oracle.ref)
        pages = len(oracle.ref)
        self.storage = torch.zeros((LAYERS, 2, pages, HEADS, oracle.page, DIM), dtype=dtype, device="cuda")
        self.storage += torch.tensor(oracle.content, device="cuda", dtype=dtype).view(1, 1, -1, 1, 1, 1)
        # layers, kinds, heads and rows differ as well
        self.mark = torch.arange(self.storage[:, :, 0].numel(), device="cuda").view(self.storage[:, :, 0].shape) % 7 * 1000
        self.storage += self.mark.unsqueeze(2).to(dtype)
        self.status = torch.full((1,), 77, dtype=torch.int32, device="cuda")
        self.workspace = torch.full((ops.pages_workspace_ints(pages),), -9, dtype=torch.int32, device="cuda")

    def check(self, oracle):
        assert self.table.tolist() == oracle.table
        assert self.lengths.tolist() == oracle.lengths
        assert self.ref.tolist() == oracle.ref
        content = torch.tensor(oracle.content, device="cuda", dtype=self.storage.dtype).view(1, 1, -1, 1, 1, 1)
        assert torch.equal(self.storage, content + self.mark.unsqueeze(2).to(self.storage.dtype))


def _state(lengths, pages, width, page, seed=0):
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    table, ref = [[-1] * width for _ in lengths], [0] * pages
    for s, length in enumerate(lengths):
        for j in range(-(-length // page)):
            table[s][j] = order.pop()
            ref[table[s][j]] = 1
    return Pages(table, list(lengths), ref, list(range(pages)), page)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _free(d, o, slots):
    from layer_streaming import ops

    ops.pages_free(_ints(slots), d.table, d.lengths, d.ref)
    o.free(slots)
    d.check(o)


def _fork(d, o, parents, children):
    from layer_streaming import ops

    ops.pages_fork(_ints(parents), _ints(children), d.table, d.lengths, d.ref, d.storage, d.status, d.workspace)
    want = o.fork(list(parents), list(children))
    assert int(d.status) == want
    d.check(o)
    return want


def _reserve(d, o, extra):
    from layer_streaming import ops

    ops.pages_reserve(_ints(extra), d.table, d.lengths, d.ref, o.page, d.status, d.workspace)
    want = o.reserve(list(extra))
    assert int(d.status) == want
    d.check(o)
    return want


def _compact(d, o, in_place):
    from layer_streaming import ops

    live = torch.full((1,), -3, dtype=torch.int32, device="cuda")
    table, ref = (d.table, d.ref) if in_place else (torch.empty_like(d.table), torch.full_like(d.ref, 5))
    ops.pages_compact(d.table, d.ref, d.storage, table, ref, live, d.workspace)
    d.table, d.ref = table, ref
    before = list(o.content)
    assert int(live) == o.compact()
    # a page that is free now holds whatever it held
    assert all(o.ref[p] or o.content[p] == before[p] for p in range(len(before)))
    d.check(o)


@pytest.mark.parametrize("page", [1, 3, 16, 64])
def test_reserve_takes_the_lowest_free_pages(cuda, page):
    o = _state([0, 5, 64, 1, 0], 300, 200, page, seed=page)
    d = Device(o)
    assert _reserve(d, o, [0, 0, 0, 0, 0]) == 0
    assert _reserve(d, o, [1, 1, 1, 1, 0]) == 0
    assert _reserve(d, o, [0, 70, 3, 0, 40]) == 0


def test_reserve_is_all_or_nothing(cuda):
    o = _state([10, 0, 30], 13, 50, 4)
    d = Device(o)
    assert _reserve(d, o, [4, 0, 6]) == 0  # 13 pages: none left
    assert _reserve(d, o, [2, 0, 0]) == 0  # fits into the last page
    assert _reserve(d, o, [1, 9, 0]) == 4
    assert _reserve(d, o, [0, 1, 0]) == 1
    assert _reserve(d, o, [0, -1, 0]) == -1
    assert _reserve(d, o, [0, 201, 0]) == -1
    assert _reserve(d, o, [0, 2 ** 31 - 1, 2 ** 31 - 1]) == -1


@pytest.mark.parametrize("page", [1, 4, 16])
@pytest.mark.parametrize("lengths", [[1, 16, 33], [64, 7, 0]])
def test_fork_shares_full_pages_and_copies_tails(cuda, page, lengths):
    o = _state(lengths + [0] * 9, 400, 90, page, seed=1)
    d = Device(o)
    assert _fork(d, o, [0, 0, 1, 2, 1], [5, 3, 4, 9, 11]) == 0
    assert _reserve(d, o, [3, 1, 0, 17, 0, 2, 0, 0, 0, 1, 0, 5]) == 0
    _free(d, o, [3, 0, 7, 3])
    assert _fork(d, o, [5, 5], [0, 3]) == 0  # a fork of a fork
    _free(d, o, list(range(12)))
    assert o.ref == [0] * 400
    assert _fork(d, o, [], []) == 0


@pytest.mark.parametrize("parents,children", [
    ([0], [12]), ([-1], [4]), ([12], [4]), ([0], [-2]), ([0], [1]), ([0, 1], [4, 4]), ([0, 4], [4, 5]), ([0], [0]),
    ([0, 1, 0], [6, 7, 1]),
])
def test_fork_refuses_wrong_slots_and_leaves_everything(cuda, parents, children):
    o = _state([5, 9, 16] + [0] * 9, 40, 10, 4)
    d = Device(o)
    assert _fork(d, o, parents, children) == -1


def test_fork_is_all_or_nothing(cuda):
    o = _state([5, 8, 3] + [0] * 5, 6, 10, 4)
    d = Device(o)
    assert _fork(d, o, [0, 1, 2], [4, 5, 6]) == 1  # one free page, two tails
    assert _fork(d, o, [0, 1], [4, 5]) == 0
    assert _fork(d, o, [2], [6]) == 1


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pages,lengths", [(1, [0]), (1, [1]), (40, [9, 30, 0, 17]), (40, [0, 0]), (3000, [900, 1200, 77]),
                                           (24, [48, 48])])
def test_compact(cuda, in_place, pages, lengths):
    page = 4
    o = _state(lengths, pages, 310, page, seed=pages)
    d = Device(o)
    _compact(d, o, in_place)
    _compact(d, o, in_place)  # a second time: nothing moves
    _reserve(d, o, [1] + [0] * (len(lengths) - 1))


@pytest.mark.parametrize("seed", range(4))
def test_random_histories(cuda, seed):
    """Long mixes of every operation, shared pages included."""

    rng = random.Random(seed)
    page, slots = rng.choice([1, 3, 8]), rng.choice([5, 40])
    o = _state([0] * slots, rng.choice([50, 700]), 40, page)
    d = Device(o)
    for _ in range(60):
        kind = rng.choice(["reserve", "fork", "free", "compact"])
        if kind == "reserve":
            _reserve(d, o, [rng.choice([0, 0, 1, rng.randint(0, 4 * page)]) for _ in range(slots)])
        elif kind == "fork":
            empty = [s for s in range(slots) if not o.lengths[s]]
            full = [s for s in range(slots) if o.lengths[s]]
            if empty and full:
                children = rng.sample(empty, rng.randint(1, min(4, len(empty))))
                _fork(d, o, [rng.choice(full) for _ in children], children)
        elif kind == "free":
            _free(d, o, [rng.randrange(slots) for _ in range(rng.randint(1, 4))])
        else:
            _compact(d, o, rng.random() < 0.5)


def test_many_sequences_and_pages(cuda):
    """More sequences and children than threads of the planning CTA, a pool that ends inside a warp's range."""

    slots, page = 2600, 2
    o = _state([(7 * s) % 4 for s in range(1300)] + [0] * 1300, 9001, 6, page)
    d = Device(o)
    parents = [s for s in range(1300) if s % 4]
    assert _fork(d, o, parents, list(range(1300, 1300 + len(parents)))) == 0
    assert _reserve(d, o, [s % 3 for s in range(slots)]) == 0
    _free(d, o, list(range(0, slots, 2)))
    _compact(d, o, True)


def test_bad_slots_and_tables_are_reported(cuda):
    from layer_streaming import _native, ops

    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    _native.check(_native.lib().cb_set_error_word(word.data_ptr()), "cb_set_error_word")
    try:
        o = _state([9, 5, 0], 20, 6, 4)
        d = Device(o)
        ops.pages_free(_ints([-1]), d.table, d.lengths, d.ref)
        assert int(word) == 621
        d.check(o)
        word.zero_()
        d.table[0, 1] = 20
        ops.pages_free(_ints([0]), d.table, d.lengths, d.ref)
        assert int(word) == 622
        assert d.ref.tolist().count(1) == 3  # page 1 of slot 0 is nobody's now; slot 1 keeps two
    finally:
        torch.cuda.synchronize()
        _native.lib().cb_set_error_word(None)


def test_refusals(cuda):
    from layer_streaming import ops

    o = _state([9, 5, 0], 20, 6, 4)
    d = Device(o)
    one = _ints([0])
    for call in (
        lambda: ops.pages_free(one.long(), d.table, d.lengths, d.ref),
        lambda: ops.pages_free(one, d.table, d.lengths[:2], d.ref),
        lambda: ops.pages_free(one, d.table.cpu(), d.lengths, d.ref),
        lambda: ops.pages_fork(one, _ints([1, 2]), d.table, d.lengths, d.ref, d.storage, d.status, d.workspace),
        lambda: ops.pages_fork(one, _ints([2]), d.table, d.lengths, d.ref[:10], d.storage, d.status, d.workspace),
        lambda: ops.pages_fork(one, _ints([2]), d.table, d.lengths, d.ref, d.storage[:, 0], d.status, d.workspace),
        lambda: ops.pages_fork(one, _ints([2]), d.table, d.lengths, d.ref, d.storage, d.status, d.workspace[:10]),
        lambda: ops.pages_fork(one, _ints([2]), d.table, d.lengths, d.ref, d.storage, d.lengths, d.workspace),
        lambda: ops.pages_reserve(_ints([1, 2]), d.table, d.lengths, d.ref, 4, d.status, d.workspace),
        lambda: ops.pages_reserve(_ints([1, 2, 3]), d.table, d.lengths, d.ref, 0, d.status, d.workspace),
        lambda: ops.pages_compact(d.table, d.ref, d.storage, d.table[:2], d.ref, d.status, d.workspace),
        lambda: ops.pages_compact(d.table, d.ref, d.storage, d.table, d.ref.long(), d.status, d.workspace),
    ):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            call()
    d.check(o)


def test_reserve_counts_what_is_missing_beyond_the_whole_pool(cuda):
    o = _state([10, 0, 30], 13, 3000, 4)
    d = Device(o)
    assert _reserve(d, o, [0, 80, 0]) == 18  # 20 pages, 2 free
    assert _reserve(d, o, [4000, 0, 9000]) == 3248
    assert _reserve(d, o, [2, 8, 2]) == 0


def test_reserve_counts_what_many_sequences_miss(cuda):
    o = _state([0] * 1500, 20, 300, 1)
    d = Device(o)
    assert _reserve(d, o, [s % 300 for s in range(1500)]) == 5 * 299 * 150 - 20
    assert _reserve(d, o, [300] * 1500) == 450000 - 20
