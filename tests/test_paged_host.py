"""Paged serving without a GPU: the binding loads and refuses, the entry points
refuse before any launch, and the oracle keeps the page bookkeeping's invariants."""

import os
import random
import subprocess
import sys

import pytest
import torch

from layer_streaming import _native, ops
from oracle import paged as oracle


def test_binding_refuses_cpu_tensors_and_other_objects():
    half = torch.zeros((2, 4, 64), dtype=torch.bfloat16)
    pool = torch.zeros((3, 2, 16, 64), dtype=torch.bfloat16)
    ints = torch.zeros((2, 3), dtype=torch.int32)
    row, byte = ints[:, 0].contiguous(), torch.zeros(64, dtype=torch.uint8)
    for call in (
        lambda: ops.paged_attention(half, pool, pool, ints, row, 1.0, half, None, byte),
        lambda: ops.paged_append(None, half, half, None, row, None, ints, None, pool, pool),
        lambda: ops.pages_free(row, ints, row, row),
        lambda: ops.pages_fork(row, row, ints, row, row, pool, row, row),
        lambda: ops.pages_reserve(row, ints, row, row, 16, row, row),
        lambda: ops.pages_compact(ints, row, pool, ints, row, row, row),
        lambda: ops.sample(half[0], None, None, None, None, row, row, None),
    ):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            call()
    with pytest.raises(TypeError, match="must be a tensor"):
        ops.pages_free(1, 2, 3, 4)
    with pytest.raises(TypeError, match="takes 8 arguments"):
        _native.binding().sample(half)
    with pytest.raises((TypeError, ValueError)):
        _native.binding().bind(1, 2)


def test_torch_operators_are_registered_for_cuda_only():
    row = torch.zeros(4, dtype=torch.int32)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.ops.cascade.pages_free(row, row.view(1, -1), row[:1], row)


def test_entry_points_refuse_before_any_launch():
    lib = _native.load_library()
    assert lib.cb_paged_append(None, 0, 0, None, 0, 0, None, 0, 0, 0, 4, 8, 2, 128, None, 128, 0, 1.0, None, None,
                               None, 1, 1, None, None, None, 1, 16, None) == 1
    assert b"null pointer" in lib.cb_last_error()
    for rotary, head_dim, dtype, message in ((24, 128, 0, b"rotary"), (128, 64, 0, b"rotary"), (0, 24, 0, b"head_dim"),
                                             (0, 64, 2, b"dtype"), (0, 1024, 1, b"head_dim")):
        assert lib.cb_paged_append(None, 0, 0, None, 0, 0, None, 0, 0, dtype, 4, 8, 2, head_dim, None, rotary, 0, 1.0,
                                   None, None, None, 1, 1, None, None, None, 1, 16, None) == 1
        assert message in lib.cb_last_error()
    attention = lambda **kw: lib.cb_paged_attention(  # noqa: E731
        None, 0, 0, None, None, kw.get("dtype", 0), kw.get("sequences", 2), kw.get("q_heads", 8), 2,
        kw.get("head_dim", 128), kw.get("pages", 9), kw.get("page_size", 16), None, kw.get("stride", 4),
        kw.get("width", 4), None, 1.0, None, None, None, 0, None)
    for kw, message in (({"dtype": 2}, b"dtype"), ({"q_heads": 7}, b"q_heads"), ({"head_dim": 80}, b"head_dim"),
                        ({"pages": 0}, b"positive"), ({"stride": 3}, b"positive"), ({}, b"null pointer"),
                        ({"page_size": 1 << 30}, b"2^31"), ({"pages": 1 << 30}, b"2^32"), ({"sequences": -1}, b"-1")):
        assert attention(**kw) == 1 and message in lib.cb_last_error(), (kw, lib.cb_last_error())
    assert attention(sequences=0) == 0  # nothing to do
    assert lib.cb_sample(None, 0, 10, 2, 0, None, None, None, None, None, None, None, None) == 1
    assert lib.cb_sample(None, 3, 10, 2, 10, None, None, None, None, None, None, None, None) == 1
    assert lib.cb_sample(None, 0, 10, 2, 10, None, None, None, None, None, None, None, None) == 1
    assert lib.cb_sample(None, 0, 10, 0, 10, None, None, None, None, None, None, None, None) == 0
    assert lib.cb_pages_free(None, 3, None, 1, 1, None, None, 1, None) == 1
    assert lib.cb_pages_reserve(None, None, 1, 1, None, None, 2000001, 16, None, None, None) == 1
    assert lib.cb_pages_workspace_ints(10) == 84 and lib.cb_pages_workspace_ints(0) == 0
    assert 0 < lib.cb_paged_attention_workspace_bytes() <= 16 << 20


def test_oracle_bookkeeping_keeps_its_invariants():
    rng = random.Random(3)
    page, slots, pages = 4, 9, 40
    o = oracle.Pages([[-1] * 8 for _ in range(slots)], [0] * slots, [0] * pages, list(range(pages)), page)
    written = {s: [] for s in range(slots)}  # what each position of a sequence holds
    mark = pages
    for _ in range(400):
        kind = rng.choice(["reserve", "fork", "free", "compact"])
        if kind == "reserve":
            extra = [rng.choice([0, 0, 1, 3]) if s % 2 or o.lengths[s] else 0 for s in range(slots)]
            if o.reserve(extra) == 0:
                for s in range(slots):  # a sequence owns the page that it writes to
                    for j in range(o.lengths[s] - extra[s], o.lengths[s]):
                        assert o.ref[o.table[s][j // page]] == 1
                        mark += 1
                        held = o.content[o.table[s][j // page]]
                        held = dict(held) if isinstance(held, dict) else {}
                        held[j % page] = mark
                        o.content[o.table[s][j // page]] = held
                        written[s].append(mark)
        elif kind == "fork":
            empty, full = [s for s in range(slots) if not o.lengths[s]], [s for s in range(slots) if o.lengths[s]]
            if empty and full:
                parent, child = rng.choice(full), rng.choice(empty)
                if o.fork([parent], [child]) == 0:
                    written[child] = list(written[parent])
        elif kind == "free":
            s = rng.randrange(slots)
            o.free([s])
            written[s] = []
        else:
            live = o.compact()
            assert all(bool(r) == (i < live) for i, r in enumerate(o.ref))
        count = [0] * pages
        for s in range(slots):
            assert [p >= 0 for p in o.table[s]] == [j < -(-o.lengths[s] // page) for j in range(8)]
            for p in o.table[s]:
                if p >= 0:
                    count[p] += 1
            assert [o.content[o.table[s][j // page]][j % page] for j in range(o.lengths[s])] == written[s]
        assert count == o.ref


def test_oracle_attention_and_rotation_on_a_small_case():
    gen = torch.Generator().manual_seed(0)
    k = torch.randn((6, 2, 4, 8), generator=gen)
    v = torch.randn((6, 2, 4, 8), generator=gen)
    q = torch.randn((2, 4, 8), generator=gen)
    table = torch.tensor([[5, 1, -1], [0, -1, -1]])
    out, lse, _, _ = oracle.attention(q, k, v, table, torch.tensor([6, 0]), 0.5)
    keys = torch.cat([k[5], k[1]], 1)[:, :6].double().repeat_interleave(2, 0)
    values = torch.cat([v[5], v[1]], 1)[:, :6].double().repeat_interleave(2, 0)
    want = torch.nn.functional.scaled_dot_product_attention(q[0].double()[:, None], keys, values, scale=0.5)[:, 0]
    torch.testing.assert_close(out[0], want)
    assert int(torch.count_nonzero(out[1])) == 0 and bool((lse[1] == -float("inf")).all())
    x = torch.randn((3, 2, 8), generator=gen)
    freq, position = torch.tensor([1.0, 0.1]), torch.tensor([0, 2, 5])
    for interleaved in (False, True):
        y = oracle.rotate(x, freq, position, interleaved)
        torch.testing.assert_close(y[0], x[0].double())
        torch.testing.assert_close(y[..., 4:], x[..., 4:].double())
        torch.testing.assert_close(y.square().sum(-1), x.double().square().sum(-1))  # a rotation
        back = oracle.rotate(y, freq, -position, interleaved)
        torch.testing.assert_close(back, x.double())


def test_the_library_builds_without_torch():
    """A user of the C interface alone needs neither Python's nor torch's headers."""

    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cascade-llm_b200", "csrc")

    def planned(python):
        run = subprocess.run(["make", "-n", "-B", "-C", csrc, "PYTHON=" + python], capture_output=True, text=True)
        assert run.returncode == 0, run.stderr
        return run.stdout

    for python in ("/nowhere/python3", sys.executable + " -S -I"):  # no Python; one without its packages
        assert "libcascade_b200.so" in planned(python) and "cascade_binding.so" not in planned(python)
    assert "libcascade_b200.so" in planned(sys.executable) and "cascade_binding.so" in planned(sys.executable)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("head_dim,group", [(64, 3), (128, 8), (128, 16)])
def test_the_cancelling_case_tells_weights_in_one_part_from_two(dtype, head_dim, group):
    q, k, v, table, lengths = oracle.cancelling_case(dtype, head_dim, group, [16, 32, 48, 2], 24)
    want, _, weight, _ = oracle.attention(q, k, v, table, lengths, 1.0)
    bound = oracle.cancelling_bound(dtype, want, weight, lengths)
    one, two = (oracle.attention_in_parts(q, k, v, table, lengths, parts) for parts in (1, 2))
    assert bool(((one - want).abs() > 2 * bound).any(-1).any(-1).all())  # planted: the rest of each weight dropped
    assert bool(((two - want).abs() <= 0.5 * bound).all())
