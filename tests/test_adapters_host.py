"""What the adapter, activation-gradient and balance entry points refuse before any device call, and the
sizes they ask for: no GPU needed."""

from __future__ import annotations

import ctypes
import random

import pytest
import torch

from crosspool_amd import _native
from crosspool_amd.adapters import AdapterPlan, AdapterWeights, interleave_gate_up_adapters
from crosspool_amd.operators import DenseAdapterLayout

BAD = _native.XP_ERROR_INVALID_ARGUMENT
# Addresses that no refused call reads.
P = 0x1000


def pool(**changes):
    fields = dict(a=P, b=P, ranks=None, scales=None, count=4, max_rank=16, input_width=64, output_width=48,
                  dtype=_native.XP_DTYPE_BF16)
    return ctypes.byref(_native.AdapterPool(**{**fields, **changes}))


def workspace(rows, backward=0, count=4, rank=16, k=64, n=48, dtype=_native.XP_DTYPE_BF16):
    return _native.library().xp_adapter_workspace_bytes(rows, count, rank, k, n, dtype, backward)


def apply(target=None, **changes):
    call = dict(ids=P, rows=8, x=0x10000, ldx=64, base=0x20000, ld_base=48, out=0x30000, ld_out=48, act=None, ws=0x40000,
                ws_bytes=1 << 30)
    call.update(changes)
    return _native.library().xp_adapter_apply(target or pool(), *call.values(), None, None)


def backward(target=None, **changes):
    call = dict(ids=P, rows=8, x=0x10000, ldx=64, grad=0x20000, ld_grad=48, base=0x30000, ld_base=64, gx=0x50000, ld_gx=64,
                ga=0x60000, gb=0x70000, ws=0x80000, ws_bytes=1 << 30)
    call.update(changes)
    return _native.library().xp_adapter_backward(target or pool(), *call.values(), None, None)


@pytest.mark.parametrize("changes", [
    dict(a=None), dict(b=None), dict(a=P + 1), dict(count=0), dict(count=1025), dict(max_rank=0), dict(max_rank=129),
    dict(input_width=0), dict(output_width=-3), dict(input_width=(1 << 22) + 1), dict(dtype=0), dict(dtype=4),
    dict(ranks=P + 2), dict(scales=P + 1),
])
def test_pools_are_checked(changes):
    assert apply(pool(**changes)) == BAD
    assert "adapter" in _native.last_error()
    assert backward(pool(**changes)) == BAD


def test_apply_refusals():
    gated = _native.ActivationDesc(function=_native.XP_ACTIVATION_SILU, gated=1, alpha=1.0)
    unknown = _native.ActivationDesc(function=9)
    ungated = _native.ActivationDesc(function=_native.XP_ACTIVATION_RELU)
    assert _native.library().xp_adapter_apply(None, P, 1, P, 64, None, 0, P, 48, None, P, 1, None, None) == BAD
    for changes in (
        dict(ids=None), dict(ids=P + 2), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(x=None), dict(x=0x10001),
        dict(ldx=63), dict(ldx=1 << 40), dict(base=0x20001), dict(ld_base=47), dict(out=None), dict(ld_out=0),
        dict(ws=None), dict(ws=0x40008), dict(ws_bytes=workspace(8) - 1), dict(act=ctypes.byref(unknown)),
        dict(out=0x10000),                                      # over the input
        dict(out=0x20010), dict(out=0x20000, ld_out=64),        # over part of the base
        dict(out=0x20000, act=ctypes.byref(ungated)),           # over the base with an activation
    ):
        assert apply(**changes) == BAD, changes
        assert _native.last_error()
    assert apply(pool(output_width=47), act=ctypes.byref(gated)) == BAD
    assert apply(rows=0, x=None, out=None, ids=None, ws=None) == _native.XP_OK


def test_backward_refusals():
    for changes in (
        dict(ids=None), dict(rows=-1), dict(x=None), dict(ldx=63), dict(grad=None), dict(ld_grad=47), dict(gx=0x50001),
        dict(ld_gx=63), dict(ga=None), dict(gb=None), dict(ga=0x60001), dict(base=0x30001), dict(ld_base=2),
        dict(gx=0x10000), dict(gx=0x20000), dict(gx=0x30010), dict(gx=0x30000, ld_gx=70), dict(ws=None),
        dict(ws_bytes=workspace(8, 1) - 1),
    ):
        assert backward(**changes) == BAD, changes
    assert backward(gx=None, ga=None, gb=None, base=None) == _native.XP_OK  # nothing asked for


def test_nothing_written_may_overlap_what_is_read():
    far = dict(a=0x1000000, b=0x2000000)
    for changes in (dict(out=0x1000010), dict(out=0x2000010), dict(out=0x40000), dict(out=P), dict(ws=0x10000),
                    dict(ws=0x20000)):
        assert apply(pool(**far), **changes) == BAD and "overlap" in _native.last_error(), changes
    for changes in (
        dict(ga=0x10000), dict(ga=0x20000), dict(ga=0x30000), dict(ga=0x50000), dict(ga=0x70000), dict(ga=0x1000010),
        dict(ga=0x2000010), dict(ga=0x80000), dict(ga=P), dict(gb=0x10010), dict(gb=0x20000), dict(gb=0x1000000),
        dict(gb=0x2000000), dict(gb=0x80000), dict(gx=0x1000000), dict(gx=0x2000000), dict(gx=0x60000), dict(gx=0x80000),
        dict(gx=P), dict(ws=0x10000), dict(ws=0x20000), dict(ws=0x30000),
    ):
        assert backward(pool(**far), **changes) == BAD and "overlap" in _native.last_error(), changes


def test_the_sorts_tables_grow_with_the_rows():
    """Runs of an adapter's rows lengthen where rows pass 256 per run: the capacity's scratch holds both sides."""

    for k, n in ((64, 64), (200, 60), (1000, 40)):
        wanted = max(1, 512 // ((k + 63) // 64 + (n + 63) // 64))
        sizes = [workspace(256 * wanted * step + extra, 1, 4, 16, k, n) for step in (1, 2, 3) for extra in (0, 1)]
        assert sizes == sorted(sizes)


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("k,n,rank,count", [(64, 48, 16, 4), (4096, 24576, 32, 32), (12288, 4096, 128, 1), (33, 5000, 3, 1024)])
def test_a_workspace_serves_every_smaller_batch(k, n, rank, count, backward):
    sizes = [1, 2, 63, 64, 65, 100, 128, 129, 1000, 2047, 8192, 8193, 33000, 70000]
    asked = [workspace(rows, backward, count, rank, k, n) for rows in sizes]
    assert asked == sorted(asked) and asked[0] > 0


def test_workspace_of_refused_sizes_is_zero():
    assert workspace(-1) == workspace(8, rank=0) == workspace(8, rank=129) == workspace(8, count=1025) == 0
    assert workspace(8, k=0) == workspace(8, n=0) == workspace(8, dtype=0) == workspace((1 << 24) + 1) == 0
    with pytest.raises(ValueError):
        AdapterPlan.prepare(row_capacity=8, adapter_count=4, max_rank=129, input_width=8, output_width=8, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        AdapterPlan.prepare(row_capacity=0, adapter_count=4, max_rank=8, input_width=8, output_width=8, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        AdapterPlan.prepare(row_capacity=8, adapter_count=4, max_rank=8, input_width=8, output_width=8, dtype=torch.float64)


def test_pools_on_the_cpu_are_refused():
    with pytest.raises(ValueError, match="GPU"):
        AdapterWeights(torch.zeros(1, 2, 3), torch.zeros(1, 4, 2))
    with pytest.raises(ValueError):
        DenseAdapterLayout(4)


def test_interleaved_gate_and_up_adapters():
    g = torch.Generator().manual_seed(0)
    gate_a, up_a = torch.randn((2, 5), generator=g), torch.randn((3, 5), generator=g)
    gate_b, up_b = torch.randn((4, 2), generator=g), torch.randn((4, 3), generator=g)
    a, b = interleave_gate_up_adapters(gate_a, gate_b, up_a, up_b)
    assert a.shape == (5, 5) and b.shape == (8, 5)
    assert torch.allclose((b @ a)[0::2], gate_b @ gate_a) and torch.allclose((b @ a)[1::2], up_b @ up_a)
    with pytest.raises(ValueError):
        interleave_gate_up_adapters(gate_a, up_b, up_a, gate_b)


def test_activation_backward_refusals():
    call = _native.library().xp_activation_backward
    silu = _native.ActivationDesc(function=_native.XP_ACTIVATION_SILU, gated=1, alpha=1.0)
    desc, bf16, pairs = ctypes.byref(silu), _native.XP_DTYPE_BF16, _native.XP_GATE_UP_INTERLEAVED
    good = dict(inputs=0x10000, grad=0x20000, out=0x30000, rows=4, width=8, dtype=bf16, order=pairs, desc=desc)
    for changes in (
        dict(desc=None), dict(rows=-1), dict(width=-1), dict(rows=1 << 31, width=2), dict(dtype=_native.XP_DTYPE_F32),
        dict(order=0), dict(inputs=None), dict(grad=None), dict(out=None), dict(out=0x30001), dict(out=0x10002),
        dict(out=0x20000),
        dict(desc=ctypes.byref(_native.ActivationDesc(function=9))),
    ):
        assert call(*{**good, **changes}.values(), None) == BAD, changes
    assert call(*{**good, "rows": 0}.values(), None) == _native.XP_OK


def test_balance_refusals():
    lib = _native.library()
    good = dict(logits=P, dtype=_native.XP_DTYPE_F32, ids=P, rows=1000, experts=16, topk=2, algorithm=1, live=None,
                coefficient=1.0, counts=P, loss=P, ws=P, ws_bytes=1 << 30)
    for changes in (
        dict(dtype=0), dict(ids=None), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(experts=0), dict(experts=1025),
        dict(topk=0), dict(topk=17), dict(algorithm=3), dict(coefficient=float("nan")), dict(coefficient=float("inf")),
        dict(counts=None), dict(loss=None), dict(logits=None), dict(logits=P + 2), dict(live=P + 1), dict(ws=None),
        dict(ws=P + 8), dict(ws_bytes=lib.xp_moe_balance_workspace_bytes(1000, 16) - 1),
    ):
        assert lib.xp_moe_balance_loss(*{**good, **changes}.values(), None) == BAD, changes
    back = dict(logits=P, dtype=_native.XP_DTYPE_BF16, counts=P, rows=10, experts=16, topk=2, algorithm=2, live=None,
                coefficient=1.0, grad_loss=None, out=P)
    for changes in (dict(logits=None), dict(counts=None), dict(out=None), dict(out=P + 1), dict(grad_loss=P + 2),
                    dict(algorithm=0), dict(dtype=9)):
        assert lib.xp_moe_balance_backward(*{**back, **changes}.values(), None) == BAD, changes
    for changes in (dict(out=P + 2), dict(counts=0x20000, out=0x20010), dict(live=0x20004, out=0x20000),
                    dict(grad_loss=0x20004, out=0x20000)):
        assert lib.xp_moe_balance_backward(*{**back, **changes}.values(), None) == BAD, changes
        assert "logits' gradient" in _native.last_error()
    assert lib.xp_moe_balance_backward(*{**back, "rows": 0}.values(), None) == _native.XP_OK
    sizes = [lib.xp_moe_balance_workspace_bytes(rows, 128) for rows in (0, 1, 256, 257, 1000, 5000, 100000)]
    assert sizes == sorted(sizes)
    assert lib.xp_moe_balance_workspace_bytes(10, 0) == lib.xp_moe_balance_workspace_bytes(-1, 8) == 0


@pytest.mark.parametrize("k,n,rank,count", [(64, 48, 16, 4), (4096, 24576, 32, 32), (33, 5000, 3, 1024)])
def test_the_workspace_of_no_rows(k, n, rank, count):
    """Gradients of no rows are cleared, with the scratch of one row; the forward needs none."""

    assert workspace(0, 0, count, rank, k, n) == 0
    assert 0 < workspace(0, 1, count, rank, k, n) <= workspace(1, 1, count, rank, k, n)
    asked = pool(a=0x100000000, b=0x200000000, count=count, max_rank=rank, input_width=k, output_width=n)
    assert backward(asked, rows=0, ids=None, x=None, ldx=0, grad=None, ld_grad=0, base=None, gx=None, ga=0x300000000,
                    gb=0x400000000, ws=0x500000000, ws_bytes=workspace(0, 1, count, rank, k, n) - 1) == BAD
    assert "smaller" in _native.last_error()


def refusal(call, k=72, n=104, **changes):
    """What a call without a workspace is refused for: "workspace" where its rows are taken."""

    assert call(pool(input_width=k, output_width=n), ws=None, **changes) == BAD
    return next(word for word in ("workspace", "overlap", "whole") if word in _native.last_error())


def test_rows_side_by_side_do_not_overlap():
    """Columns of one tensor of 600 bf16 columns, at byte offsets of twice their first."""

    base = 0x1000000
    wide = dict(rows=300, x=base, ldx=600, base=base + 144, ld_base=600, out=base + 352, ld_out=600)
    assert refusal(apply, **wide) == "workspace"
    assert refusal(apply, **{**wide, "out": base + 350}) == "whole"            # the base's last column
    assert refusal(apply, **{**wide, "out": base + 1200 - 206}) == "overlap"   # one column into the next rows of x
    assert refusal(apply, **{**wide, "out": base + 1200 - 208}) == "workspace"
    assert refusal(apply, **{**wide, "out": base - 206, "base": None}) == "overlap"
    assert refusal(apply, **{**wide, "out": base - 208, "base": None}) == "workspace"
    # Past the last row, and before the first, where no row of x follows or precedes.
    last = base + 299 * 1200
    assert refusal(apply, **{**wide, "out": last + 142, "base": None}) == "overlap"
    assert refusal(apply, **{**wide, "out": last + 144, "base": None}) == "workspace"
    assert refusal(apply, **{**wide, "out": base - 299 * 1200 - 206, "base": None}) == "overlap"
    assert refusal(apply, **{**wide, "out": base - 299 * 1200 - 208, "base": None}) == "workspace"
    # Every other row, and rows of another stride.
    assert refusal(apply, **{**wide, "ldx": 1200, "out": base + 1200, "ld_out": 1200, "base": None}) == "workspace"
    assert refusal(apply, **{**wide, "out": base + 1200, "ld_out": 1200, "base": None}) == "overlap"
    assert refusal(apply, **{**wide, "out": base + 144, "ld_out": 1200, "base": None}) == "workspace"
    # One row.
    assert refusal(apply, **{**wide, "rows": 1, "out": base + 142, "base": None}) == "overlap"
    assert refusal(apply, **{**wide, "rows": 1, "out": base + 144, "base": None}) == "workspace"
    back = dict(rows=300, x=base, ldx=600, grad=base + 144, ld_grad=600, base=base + 352, ld_base=600, gx=base + 496,
                ld_gx=600, ga=0x4000000, gb=0x5000000)
    assert refusal(backward, **back) == "workspace"
    assert refusal(backward, **{**back, "gx": base + 494}) == "whole"
    assert refusal(backward, **{**back, "gx": base + 350, "base": None}) == "overlap"


def test_rows_overlap_where_they_share_a_byte():
    """Rows of any strides and places, against the bytes counted one by one."""

    rng = random.Random(0)
    found = []
    for _ in range(3000):
        k, n, rows = rng.randint(1, 5), rng.randint(1, 5), rng.randint(1, 6)
        ldx = k + rng.choice((0, 1, rng.randint(0, 20)))
        ld_out = n + rng.choice((0, rng.randint(0, 20))) if rng.random() < 0.4 else max(ldx, n)
        start = 2 * rng.randint(-60, 60)
        read = {i * ldx * 2 + byte for i in range(rows) for byte in range(2 * k)}
        written = {start + i * ld_out * 2 + byte for i in range(rows) for byte in range(2 * n)}
        found.append(bool(read & written))
        reason = refusal(apply, k, n, rows=rows, x=0x10000, ldx=ldx, base=None, out=0x10000 + start, ld_out=ld_out)
        assert reason == ("overlap" if found[-1] else "workspace"), (k, n, rows, ldx, ld_out, start)
    assert 500 < sum(found) < 2500


def test_nothing_written_may_overlap_the_pools_tables_or_the_workspace():
    """The workspace over the pool or the ids, anything over ranks and scales, and the fault word over anything."""

    tables = dict(a=0x100000000, b=0x200000000, ranks=0x300000000, scales=0x400000000)
    size = workspace(8)
    for at in (0x100000000, 0x200000000, 0x300000000, 0x400000000, P):
        for shift in (0, 0x10 - size // 16 * 16):   # its first bytes over the table, or its last
            assert apply(pool(**tables), ws=at + shift) == BAD and "overlap" in _native.last_error(), (at, shift)
            assert backward(pool(**tables), ws=at + shift) == BAD and "overlap" in _native.last_error(), (at, shift)
    for at in (0x300000000, 0x300000008, 0x400000000, 0x40000000c):
        assert apply(pool(**tables), out=at) == BAD and "overlap" in _native.last_error()
        for name in ("gx", "ga", "gb"):
            assert backward(pool(**tables), **{name: at}) == BAD and "overlap" in _native.last_error(), name

    def with_fault(call, word):
        descriptor = _native.AdapterPool(**dict(count=4, max_rank=16, input_width=64, output_width=48,
                                                dtype=_native.XP_DTYPE_BF16, **tables))
        function = "xp_adapter_apply" if call is apply else "xp_adapter_backward"
        given = ([P, 8, 0x10000, 64, 0x20000, 48, 0x30000, 48, None, 0x40000] if call is apply
                 else [P, 8, 0x10000, 64, 0x20000, 48, 0x30000, 64, 0x50000, 64, 0x60000, 0x70000, 0x80000])
        return getattr(_native.library(), function)(ctypes.byref(descriptor), *given, 1 << 30, word, None)

    for word in (P, 0x10000, 0x20004, 0x30000, 0x40000, *tables.values()):
        assert with_fault(apply, word) == BAD and "overlap" in _native.last_error(), hex(word)
    for word in (P + 4, 0x10000, 0x20004, 0x30000, 0x50000, 0x60000, 0x70000, 0x80000, *tables.values()):
        assert with_fault(backward, word) == BAD and "overlap" in _native.last_error(), hex(word)


def test_nothing_of_the_balance_loss_may_overlap():
    lib = _native.library()
    good = dict(logits=0x1000000, dtype=_native.XP_DTYPE_F32, ids=0x2000000, rows=1000, experts=16, topk=2, algorithm=1,
                live=0x3000000, coefficient=1.0, counts=0x4000000, loss=0x5000000, ws=0x6000000, ws_bytes=1 << 30)
    for changes in (
        dict(ws=0x1000000), dict(ws=0x1000000 + 63984), dict(ws=0x2000000), dict(ws=0x3000000), dict(ws=0x4000000),
        dict(ws=0x5000000), dict(counts=0x1000000), dict(counts=0x2000000 + 7996), dict(counts=0x3000000 - 60),
        dict(counts=0x5000000 - 4), dict(loss=0x1000000 + 63996), dict(loss=0x2000000), dict(loss=0x3000000),
        dict(loss=0x4000000 + 60), dict(rows=10, ws=None, ws_bytes=0, counts=0x2000000),
        dict(logits=None, loss=None, counts=0x2000000),
    ):
        assert lib.xp_moe_balance_loss(*{**good, **changes}.values(), None) == BAD, changes
        assert "overlap" in _native.last_error(), changes


def test_the_fault_words_alignment():
    lib, far = _native.library(), pool(a=0x1000000, b=0x2000000)
    assert lib.xp_adapter_apply(far, P, 8, 0x10000, 64, 0x20000, 48, 0x30000, 48, None, 0x40000, 1 << 30, 0x3000002, None) == BAD
    assert "aligned" in _native.last_error()
    assert lib.xp_adapter_backward(far, P, 8, 0x10000, 64, 0x20000, 48, None, 0, 0x50000, 64, None, None, 0x80000, 1 << 30,
                                   0x3000001, None) == BAD
    assert "aligned" in _native.last_error()


def test_transposes_have_room_for_the_adapters_with_rows_only():
    """Weights of 1024 adapters of rank 8 (padded to 16) are 940 MB; a batch of one row uses one of them."""

    k, n = 4096, 24576
    one = 16 * (k + n) * 2
    for rows in (1, 2, 40, 64):
        # Beside the transposes: partial sums and coefficients of a tile, tables of ints of the pool.
        assert rows * one < workspace(rows, 1, 1024, 8, k, n) < (rows + 1) * one + 512 * 1024, rows
    assert workspace(5000, 1, 1024, 8, k, n) > 1024 * one
    # Up to 32 adapters every one has its place.
    assert workspace(1, 1, 32, 8, k, n) > 32 * one
