"""esgd.ops and include/esgd_ops.h without a device: what they refuse, and with what message.
The operators' results are in test_ops_gpu.py."""
import ctypes as C

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from esgd import _lib, ops

F, BF, H = _lib.FLOAT, _lib.BF16, ops.HALF


def _refuses(match, fn, *args, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*args, **kw)


def test_no_cpu_path():
    w, t = torch.zeros(5, 4), torch.zeros(3, dtype=torch.long)
    _refuses("no CPU path", ops.embedding, w, t)
    _refuses("no CPU path", ops.embedding, w.requires_grad_(), t)
    _refuses("no CPU path", ops.embedding_grad, torch.zeros(3, 4), t, 5)
    _refuses("no CPU path", ops.expert_sort, torch.zeros(3, 2, dtype=torch.int32), 4)
    order = ops.ExpertOrder(torch.zeros(5, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32), 4)
    _refuses("no CPU path", ops.expert_dispatch, torch.zeros(3, 4), order)
    _refuses("no CPU path", ops.expert_dispatch_grad, torch.zeros(6, 4), order)
    _refuses("no CPU path", ops.expert_combine, torch.zeros(6, 4), torch.zeros(3, 2), order)
    _refuses("no CPU path", ops.expert_combine_grad, torch.zeros(3, 4), torch.zeros(6, 4), torch.zeros(3, 2), order)
    z, top, i = torch.zeros(2, 7), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.long)
    _refuses("no CPU path", ops.distill_loss, z, top, i)
    _refuses("no CPU path", ops.distill_loss_grad, z, top, i, torch.ones(2))


def test_embedding_refusals():
    w, t = torch.zeros(5, 4), torch.zeros(3, dtype=torch.long)
    _refuses("float64", ops.embedding, w.double(), t)
    _refuses("dimensions", ops.embedding, w[0], t)
    _refuses("int32 or int64", ops.embedding, w, t.float())
    _refuses("int32 or int64", ops.embedding, w, t.to(torch.int16))
    _refuses("its own type", ops.embedding, w.bfloat16(), t, dtype=torch.float32)
    _refuses("its own type", ops.embedding, w, t, dtype=torch.float64)
    g = torch.zeros(3, 4)
    _refuses("a row for each", ops.embedding_grad, g, t[:2], 5)
    _refuses("a row for each", ops.embedding_grad, g[0], t, 5)
    _refuses("negative", ops.embedding_grad, g, t, -1)
    _refuses("needs out", ops.embedding_grad, g, t, 5, accumulate=True)
    _refuses("contiguous", ops.embedding_grad, g, t, 5, out=torch.zeros(4, 4))
    _refuses("contiguous", ops.embedding_grad, g, t, 5, out=torch.zeros(4, 5).t())
    _refuses("dtype says", ops.embedding_grad, g, t, 5, out=torch.zeros(5, 4), dtype=torch.bfloat16)
    _refuses("that type or float32", ops.embedding_grad, g, t, 5, dtype=torch.bfloat16)
    _refuses("that type or float32", ops.embedding_grad, g, t, 5, out=torch.zeros(5, 4, dtype=torch.float64))
    with pytest.raises(_lib.EsgdError, match="too many"):
        ops.embedding_grad(g, t, 1 << 31)


def test_expert_refusals():
    e = torch.zeros(3, 2, dtype=torch.int32)
    _refuses("int32 or int64", ops.expert_sort, e.float(), 4)
    _refuses("neither", ops.expert_sort, e[None], 4)
    _refuses("neither", ops.expert_sort, e[:, :0], 4)
    for bad in (0, -1, 1 << 24):
        with pytest.raises(_lib.EsgdError):
            ops.expert_sort(e, bad)
    order = ops.ExpertOrder(torch.zeros(5, dtype=torch.int32), e, 4)
    x, y, w = torch.zeros(3, 4), torch.zeros(6, 4), torch.zeros(3, 2)
    _refuses("rows for 3 tokens", ops.expert_dispatch, y, order)
    _refuses("float64", ops.expert_dispatch, x.double(), order)
    _refuses("dimensions", ops.expert_dispatch, x[None], order)
    _refuses("rows for 3 tokens", ops.expert_dispatch_grad, x, order)
    _refuses("rows for 3 tokens", ops.expert_combine, x, w, order)
    _refuses("weights", ops.expert_combine, y, w[:, :1], order)
    _refuses("weights", ops.expert_combine, y, w.long(), order)
    _refuses("rows of 4", ops.expert_combine_grad, x[:, :3], y, w, order)
    _refuses("rows of 4", ops.expert_combine_grad, x.bfloat16(), y, w, order)
    _refuses("rows for 3 tokens", ops.expert_combine_grad, y, y, w, order)


def test_distill_refusals():
    z, t, i, g = torch.zeros(2, 7), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.long), torch.ones(2)
    _refuses("float64", ops.distill_loss, z.double(), t, i)
    _refuses("no vocabulary", ops.distill_loss, z[:, :0], t, i)
    _refuses("go together", ops.distill_loss, z, t[:1], i[:1])
    _refuses("go together", ops.distill_loss, z, t, i[:, :2])
    _refuses("go together", ops.distill_loss, z, t[0], i[0])
    _refuses("int32 or int64", ops.distill_loss, z, t, i.float())
    big = torch.zeros(2, ops.TOP_MAX + 1)
    _refuses("at most", ops.distill_loss, z, big, big.long())
    for bad in (0.0, -1.0, float("nan"), float("inf"), 1e-5, 1e5):
        _refuses("temperature", ops.distill_loss, z, t, i, bad)
    _refuses("float32 is needed", ops.distill_loss_grad, z, t, i, g.bfloat16())
    _refuses("row_grad", ops.distill_loss_grad, z, t, i, torch.ones(3))


def test_c_entry_points_refuse_before_they_look_for_a_device():
    # the C ABI by itself: null and misaligned pointers, sizes, types, short work memory
    h = _lib.lib()
    p, bad = C.c_void_p(0x10000), _lib.INVALID_ARG
    z = C.c_size_t()
    assert h.esgd_embedding(F, p, 4, 5, 4, 16, p, 3, 1.0, F, p, 4, None) == bad and "16 bits" in _lib.last_error()
    assert h.esgd_embedding(BF, p, 4, 5, 4, 64, p, 3, 1.0, F, p, 4, None) == bad
    assert h.esgd_embedding(F, p, 4, 5, 4, 64, None, 3, 1.0, F, p, 4, None) == bad
    assert h.esgd_embedding(F, p, 4, 5, 4, 64, p, 3, 1.0, F, p, 3, None) == bad
    assert h.esgd_embedding(F, p, 4, -1, 4, 64, p, 3, 1.0, F, p, 4, None) == bad
    assert h.esgd_embedding_grad_work(10, 5, 4, None) == bad
    assert h.esgd_embedding_grad_work(1 << 31, 5, 4, C.byref(z)) == bad
    assert h.esgd_embedding_grad_work(10, 5, 4, C.byref(z)) == 0 and z.value > 0
    args = [F, p, 4, 10, 4, 64, p, -1, 1.0, F, p, 5, 0, p, z.value, None]
    assert h.esgd_embedding_grad(*args[:14], z.value - 1, None) == bad and "needed" in _lib.last_error()
    assert h.esgd_embedding_grad(*args[:13], C.c_void_p(0x10008), z.value, None) == bad
    assert h.esgd_embedding_grad(99, *args[1:]) == bad
    assert h.esgd_embedding_grad(BF, *args[1:9], H, *args[10:]) == bad
    assert h.esgd_expert_sort_work(10, 0, C.byref(z)) == bad
    assert h.esgd_expert_sort_work(10, 4, C.byref(z)) == 0
    assert h.esgd_expert_sort(32, p, 5, 0, 4, p, p, p, z.value, None) == bad
    assert h.esgd_expert_sort(8, p, 5, 2, 4, p, p, p, z.value, None) == bad
    assert h.esgd_expert_sort(32, p, 5, 2, 4, p, p, p, 0, None) == bad
    assert h.esgd_expert_sort(32, p, 5, 2, 4, None, p, p, z.value, None) == bad
    assert h.esgd_expert_dispatch(_lib.DOUBLE, p, 4, 5, 2, 4, p, p, None) == bad
    assert h.esgd_expert_dispatch(F, p, 4, 1 << 31, 2, 4, p, p, None) == bad
    assert h.esgd_expert_dispatch_grad(F, p, -4, 5, 2, 4, p, p, None) == bad
    assert h.esgd_expert_combine(F, p, 4, 5, 2, 4, p, None, p, None) == bad
    assert h.esgd_expert_combine_grad(F, p, 4, p, 4, 5, 2, 4, p, p, p, None, None) == bad
    row = [F, p, 7, 2, 7, F, p, 64, p, 3, 1.0]
    assert h.esgd_distill_work(2, 0, C.byref(z)) == bad
    assert h.esgd_distill_loss(*row[:10], 0.0, p, p, None, 0, None) == bad
    assert h.esgd_distill_loss(*row[:9], ops.TOP_MAX + 1, 1.0, p, p, None, 0, None) == bad
    assert h.esgd_distill_loss(*row, p, C.c_void_p(0x10004), None, 0, None) == bad and "16-byte" in _lib.last_error()
    assert h.esgd_distill_grad(*row, None, p, 1, p, None) == bad
    assert h.esgd_distill_loss_grad(*row, None, 1, p, p, p, None, 0, None) == bad
    assert h.esgd_distill_work(2, 1 << 20, C.byref(z)) == 0 and z.value > 0
    assert h.esgd_distill_loss(F, p, 1 << 20, 2, 1 << 20, F, p, 64, p, 3, 1.0, p, p, p, z.value - 1, None) == bad
    if _lib.device_count() == 0:   # a sound call: no device
        assert h.esgd_embedding(F, p, 4, 5, 4, 64, p, 3, 1.0, F, p, 4, None) == _lib.NO_DEVICE
        assert h.esgd_distill_loss(*row, p, p, None, 0, None) == _lib.NO_DEVICE


def test_empty_calls_need_no_device():
    # nothing to do is no error, with null pointers too (the C conventions of esgd.h)
    h = _lib.lib()
    assert h.esgd_embedding(F, None, 4, 5, 4, 64, None, 0, 1.0, F, None, 4, None) == 0
    assert h.esgd_expert_dispatch(F, None, 4, 0, 2, 4, None, None, None) == 0
    assert h.esgd_expert_combine(F, None, 4, 0, 2, 4, None, None, None, None) == 0
    assert h.esgd_distill_loss(F, None, 7, 0, 7, F, None, 64, None, 3, 1.0, None, None, None, 0, None) == 0


def test_negative_padding_index_is_refused():
    # nn.Embedding counts it from the table's end; here tokens outside the table are padding already
    w, t = torch.zeros(5, 4), torch.zeros(3, dtype=torch.long)
    _refuses("negative", ops.embedding, w, t, padding_index=-1)
    _refuses("negative", ops.embedding_grad, torch.zeros(3, 4), t, 5, padding_index=-1)


def test_views_with_a_sign_to_come_are_refused():
    # their memory holds the values of the other sign
    w = torch.view_as_complex(torch.ones(5, 4, 2)).conj().imag
    assert w.is_neg()
    _refuses("resolve_neg", ops.embedding, w, torch.zeros(3, dtype=torch.long))
    _refuses("resolve_neg", ops.distill_loss, w, torch.zeros(5, 3), torch.zeros(5, 3, dtype=torch.long))
    z, top, i = torch.zeros(5, 7), torch.zeros(5, 3), torch.zeros(5, 3, dtype=torch.long)
    _refuses("resolve_neg", ops.distill_loss_grad, z, top, i, w[:, 0])


def test_embedding_grad_refuses_an_out_that_shares_memory():
    buf, t = torch.zeros(40), torch.zeros(5, dtype=torch.long)
    _refuses("shares memory with grad", ops.embedding_grad, buf[:20].view(5, 4), t, 5, out=buf[:20].view(5, 4))
    _refuses("shares memory with grad", ops.embedding_grad, buf[:20].view(5, 4), t, 5, out=buf[16:36].view(5, 4))
    _refuses("shares memory with tokens", ops.embedding_grad, torch.zeros(5, 4), t, 2,
             out=t.view(torch.float32)[:8].view(2, 4))
    _refuses("no CPU path", ops.embedding_grad, buf[:20].view(5, 4), t, 5, out=buf[20:].view(5, 4))


def test_embedding_grad_refuses_an_out_among_the_rows_it_reads():
    # rows that stand apart are read where they lie: the table's zeros must not go there
    buf, t = torch.zeros(10, 8), torch.zeros(10, dtype=torch.long)
    flat = buf.view(-1)
    _refuses("shares memory with grad", ops.embedding_grad, buf[:, :4], t, 10, out=flat[:40].view(10, 4))
    _refuses("shares memory with grad", ops.embedding_grad, buf[:, :4], t, 1, out=flat[75:79].view(1, 4))
    _refuses("shares memory with grad", ops.embedding_grad, buf[::2], t[:5], 5, out=buf[:5])
    _refuses("shares memory with grad", ops.embedding_grad, buf[0].expand(10, 8), t, 10, out=buf)
    _refuses("shares memory with grad", ops.embedding_grad, buf[:, None, 2:5], t[:, None], 2, out=flat[1:7].view(2, 3))
    # a copy of the caller's that names the same memory in a storage of its own
    alias = torch.frombuffer(memoryview(buf.numpy()).cast("B"), dtype=torch.float32)
    _refuses("shares memory with grad", ops.embedding_grad, buf[:, :4], t, 10, out=alias[:40].view(10, 4))
    # between the rows, behind them and in memory of its own: sound
    for rows, out in ((1, flat[4:8].view(1, 4)), (1, flat[76:80].view(1, 4)), (2, torch.zeros(2, 4)), (0, flat[:0].view(0, 4))):
        _refuses("no CPU path", ops.embedding_grad, buf[:, :4], t, rows, out=out)
    # what is copied before the table is zeroed
    _refuses("no CPU path", ops.embedding_grad, buf[:, ::2], t, 10, out=flat[:40].view(10, 4))


def _every_call():
    """Each operator on small tensors that it accepts but for their device, as (operator, its
    arguments, the places of the floating tensors among them)."""
    w, t = torch.zeros(5, 4), torch.zeros(3, dtype=torch.long)
    order = ops.ExpertOrder(torch.zeros(5, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32), 4)
    x, y, k = torch.zeros(3, 4), torch.zeros(6, 4), torch.zeros(3, 2)
    z, top, i = torch.zeros(2, 7), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.long)
    return [(ops.embedding, (w, t), (0,)), (ops.embedding_grad, (x, t, 5), (0,)),
            (ops.expert_dispatch, (x, order), (0,)), (ops.expert_dispatch_grad, (y, order), (0,)),
            (ops.expert_combine, (y, k, order), (0, 1)), (ops.expert_combine_grad, (x, y, k, order), (0, 1, 2)),
            (ops.distill_loss, (z, top, i), (0, 1)), (ops.distill_loss_grad, (z, top, i, torch.ones(2)), (0, 1, 3))]


def test_tangents_of_forward_mode_are_refused():
    # there is no forward-mode derivative: an answer without a tangent would say that it is zero
    for fn, args, floats in _every_call():
        _refuses("no CPU path", fn, *args)
        for at in floats:
            for wants_grad in (False, True):
                with forward_ad.dual_level():
                    primal = args[at].clone().requires_grad_(wants_grad)
                    dual = forward_ad.make_dual(primal, torch.ones_like(primal))
                    _refuses("tangent", fn, *args[:at], dual, *args[at + 1:])

            def of_one(x, fn=fn, args=args, at=at):
                return fn(*args[:at], x, *args[at + 1:])

            with pytest.raises(ValueError, match="tangent"):
                torch.func.jvp(of_one, (args[at],), (torch.ones_like(args[at]),))
    out = torch.zeros(5, 4)
    with forward_ad.dual_level():
        _refuses("tangent", ops.embedding_grad, torch.zeros(3, 4), torch.zeros(3, dtype=torch.long), 5,
                 out=forward_ad.make_dual(out, out))


def test_embedding_grad_refuses_an_out_with_a_sign_to_come():
    # a negated view is contiguous, but its memory is read with the other sign
    g, t = torch.zeros(3, 4), torch.zeros(3, dtype=torch.long)
    out = torch._neg_view(torch.ones(5, 4))
    assert out.is_contiguous() and out.is_neg()
    for accumulate in (False, True):
        _refuses("resolve_neg", ops.embedding_grad, g, t, 5, out=out, accumulate=accumulate)


def test_embedding_grad_refuses_an_out_that_requires_a_gradient():
    # as torch's own calls with out=: autograd would not know of the write
    g, t = torch.zeros(3, 4), torch.zeros(3, dtype=torch.long)
    leaf = torch.ones(5, 4, requires_grad=True)
    for out in (leaf, leaf * 2):
        for accumulate in (False, True):
            _refuses("requires a gradient", ops.embedding_grad, g, t, 5, out=out, accumulate=accumulate)
            with torch.no_grad():
                _refuses("no CPU path", ops.embedding_grad, g, t, 5, out=out, accumulate=accumulate)


def test_tensors_in_the_place_of_numbers_are_refused():
    # their gradient would be lost, and on a GPU the call would wait for their value
    w, t, e = torch.zeros(5, 4), torch.zeros(3, dtype=torch.long), torch.zeros(3, 2, dtype=torch.int32)
    z, top, i = torch.zeros(2, 7), torch.zeros(2, 3), torch.zeros(2, 3, dtype=torch.long)
    for x in (torch.tensor(2.0), torch.tensor(2.0, requires_grad=True), torch.nn.Parameter(torch.ones(1))):
        for weight in (w, torch.zeros(5, 4, requires_grad=True)):
            _refuses("scale is a tensor", ops.embedding, weight, t, x)
        _refuses("scale is a tensor", ops.embedding_grad, torch.zeros(3, 4), t, 5, x)
        for logits in (z, torch.zeros(2, 7, requires_grad=True)):
            _refuses("temperature is a tensor", ops.distill_loss, logits, top, i, x)
        _refuses("temperature is a tensor", ops.distill_loss_grad, z, top, i, torch.ones(2), x)
    one = torch.tensor(1)
    _refuses("padding_index is a tensor", ops.embedding, w, t, padding_index=one)
    _refuses("padding_index is a tensor", ops.embedding_grad, torch.zeros(3, 4), t, 5, padding_index=one)
    _refuses("num_rows is a tensor", ops.embedding_grad, torch.zeros(3, 4), t, one)
    _refuses("num_experts is a tensor", ops.expert_sort, e, one)
    for number in (2, 2.0, True, np.float32(2.0), np.int64(2)):   # any other number will do
        _refuses("no CPU path", ops.embedding, w, t, number)
        _refuses("no CPU path", ops.distill_loss, z, top, i, number)


def test_embedding_grad_asks_for_the_work_memory_that_it_uses():
    # the sort's share, which a width of 0 shows alone, and two fp32 rows for every tile of sorted
    # rows.  Tiles are 64 rows, halved down to 8 until their loads -- lane_bytes for each 64 * columns
    # of a tile -- are 2048 waves' of 16 bytes; (columns, lane_bytes) of the gradient's and table's types:
    types = {(F, F): (4, 16), (BF, F): (4, 8), (BF, BF): (8, 16)}
    h, z = _lib.lib(), C.c_size_t()

    def asked(n, width):
        assert h.esgd_embedding_grad_work(n, 1000, width, C.byref(z)) == 0
        return z.value

    def tiles(n, width, columns, lane_bytes):
        chunks, per = -(-width // (64 * columns)), 64
        while per > 8 and -(-n // per) * chunks * lane_bytes < 2048 * 16:
            per //= 2
        return -(-n // per)

    sizes = [(n, w) for n in (1, 7, 8, 9, 4095, 4096, 32767, 32768, 65536, 65537, 131072, 262144, 1048576)
             for w in (1, 255, 256, 257, 512, 513, 1000, 1024, 4096)]
    for n in (8192, 16384, 16385, 32768, 32769):   # both sides of every change of the tile's rows
        sizes += [(n * k + d, w) for k in (1, 2, 4) for d in (-1, 0, 1) for w in (256, 512, 1024)]
    for n, w in sizes:
        most = max(tiles(n, w, *t) for t in types.values())
        assert asked(n, w) - asked(n, 0) == most * 2 * w * 4, (n, w)
    assert asked(131072, 1024) < 20 << 20   # 130 MiB with room for tiles of 8
