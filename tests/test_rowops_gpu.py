"""The row operators on the GPU against their plain 64-bit forms (oracle/rowops_oracle.py), whose bounds count roundings."""
import copy
import os

import pytest
import torch

from oracle import rowops_oracle as ro

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
INF = float("inf")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ops():
    from hyc_lora_b200 import rowops
    return rowops


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=_gen(seed)) * scale).to(dtype)


def _rng(seed=11, call=5):
    return torch.tensor([seed, call], dtype=torch.int64)


def _offset(t, elements):
    """A contiguous CUDA copy of ``t`` that starts ``elements`` elements behind an aligned address."""
    buf = torch.empty(t.numel() + elements, dtype=t.dtype, device="cuda")
    out = buf[elements:].view(t.shape)
    out.copy_(t)
    return out


def _near(got, want, bound, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, torch.zeros_like(got), (got - want).abs())
    bad = ~(off <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {off[bad].max().item():.3e} " \
                                f"where {bound.expand_as(off)[bad].min().item():.3e} is allowed"


# ---------------------------------------------------------------------------------------------------- dropout

@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(1,), (3,), (1, 4), (3, 5), (7, 8), (2, 3, 16), (5, 1001), (64, 768), (3, 4096), (2049, 129)])
@pytest.mark.parametrize("p", [0.1, 0.5])
@pytest.mark.parametrize("with_residual", [False, True])
def test_dropout_matches_the_plain_form(ops, dtype, shape, p, with_residual):
    x = _randn(shape, dtype, 1, 3.0)
    res = _randn(shape, dtype, 2) if with_residual else None
    rng = _rng(seed=-2 ** 62 + 17, call=2 ** 40 + 3)
    want, bound = ro.dropout(x, p, ro.keep_mask(-2 ** 62 + 17, 2 ** 40 + 3, p, shape), res)
    got = ops.dropout(x.cuda(), p, rng.cuda(), residual=None if res is None else res.cuda())
    assert got.dtype == dtype and got.is_contiguous()
    _near(got, want, bound)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("p", [0.0, 1.0, 1.0 - 2.0 ** -40, 2.0 ** -40])
def test_dropout_at_the_ends_of_its_range(ops, dtype, p):
    x = _randn((9, 50), dtype, 3)
    x[0, :4] = torch.tensor([INF, -INF, float("nan"), 1.0])
    got = ops.dropout(x.cuda(), p, _rng().cuda(), residual=torch.ones_like(x).cuda()).cpu()
    if p > 0.5:
        assert torch.equal(got, torch.ones_like(x))          # nothing is kept, and nothing of x is seen
    else:
        want = (x.double() + 1).to(dtype)
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("offsets", [(1, 0), (0, 1), (3, 5), (4, 4)])
def test_dropout_of_unaligned_and_strided_tensors(ops, dtype, offsets):
    x, res = _randn((33, 40), dtype, 4), _randn((33, 40), dtype, 5)
    keep = ro.keep_mask(11, 5, 0.3, x.shape)
    want, bound = ro.dropout(x, 0.3, keep, res)
    _near(ops.dropout(_offset(x, offsets[0]), 0.3, _rng().cuda(), residual=_offset(res, offsets[1])), want, bound, "offset")
    wide = torch.full((33, 56), 99.0, dtype=dtype, device="cuda")
    for first in (0, 8, 3):
        view = wide[:, first:first + 40]
        view.copy_(x)
        _near(ops.dropout(view, 0.3, _rng().cuda(), residual=res.cuda()), want, bound, f"columns from {first}")
        _near(ops.dropout(res.cuda(), 0.3, _rng().cuda(), residual=view), *ro.dropout(res, 0.3, keep, x), "strided residual")
    turned = x.t().contiguous().cuda().t()                   # elements of a row apart: copied
    _near(ops.dropout(turned, 0.3, _rng().cuda()), *ro.dropout(x, 0.3, keep))
    one = x[:1].expand(33, 40)
    _near(ops.dropout(x[:1].cuda().expand(33, 40), 0.3, _rng().cuda()), *ro.dropout(one, 0.3, keep), "one row, seen 33 times")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("p", [0.1, 0.05, 0.3])
@pytest.mark.parametrize("rows,cols,offset", [(64, 768, 0), (3, 1001, 0), (64, 768, 1), (3000, 2048, 0)])
def test_kept_values_are_rounded_before_the_residual_is_added(ops, dtype, p, rows, cols, offset):
    """Each of product and sum is one IEEE operation, so the results are known to the bit.  Half of the residuals are what the
    kept value is taken from (sums of exactly zero in fp32), and the inputs have few digits (sums on ties of bf16)."""
    x = torch.randint(-255, 256, (rows, cols), generator=_gen(1)).float().mul_(9.0 / 64).to(dtype)
    scale = torch.tensor(1.0 / (1.0 - p), dtype=F32)
    away = torch.rand((rows, cols), generator=_gen(2)) < 0.5
    res = torch.where(away, -(x.float() * scale), _randn((rows, cols), F32, 3, 8.0)).to(dtype)
    keep = ro.keep_mask(11, 5, p, x.shape)
    z = torch.where(keep, x.float() * scale, torch.zeros(())) + res.float()
    if dtype == F32:
        assert bool((z[away & keep] == 0).all())
    got = ops.dropout(_offset(x, offset), p, _rng().cuda(), residual=_offset(res, offset))
    assert torch.equal(got.cpu(), z.to(dtype))
    out = ops.layer_norm(_offset(x, offset), None, None, residual=_offset(res, offset), p=p, rng=_rng().cuda())
    assert torch.equal(out.z.cpu(), z.to(dtype))


def test_dropout_of_nothing(ops):
    for shape in ((0,), (0, 8), (5, 0), (2, 0, 3)):
        x = torch.empty(shape, dtype=BF16, device="cuda")
        assert ops.dropout(x, 0.1, _rng().cuda(), residual=x).shape == shape


def test_dropout_writes_its_own_elements_only(ops):
    """The output sits between flanks of the allocator's: checked through the C entry point."""
    import ctypes as C
    from hyc_lora_b200 import _lib
    for n in (1, 3, 5, 1003):
        for lead in (0, 1, 8):
            x = _randn((n,), BF16, n).cuda()
            rng = _rng().cuda()
            buf = torch.full((n + 48,), -7.0, dtype=BF16, device="cuda")
            a = _lib.HycDropoutArgs()
            a.rows, a.cols, a.dtype, a.p = 1, n, _lib.HYC_BF16, 0.5
            a.x, a.y, a.rng = x.data_ptr(), buf[16 + lead:].data_ptr(), rng.data_ptr()
            assert _lib.lib.hyc_dropout(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
            torch.cuda.synchronize()
            assert bool((buf[:16 + lead] == -7).all()) and bool((buf[16 + lead + n:] == -7).all())
            _near(buf[16 + lead:16 + lead + n], *ro.dropout(x.cpu(), 0.5, ro.keep_mask(11, 5, 0.5, (n,))))


def test_dropout_beyond_32_bit_offsets(ops):
    n = 2 ** 32 + 4099
    x = torch.ones(n, dtype=BF16, device="cuda")
    y = ops.dropout(x, 0.25, _rng().cuda())
    for first in (0, 2 ** 31 - 64, 2 ** 32 - 64, n - 4099):
        keep = ro.keep_mask(11, 5, 0.25, (128,), first=first)
        want, bound = ro.dropout(torch.ones(128, dtype=BF16), 0.25, keep)
        _near(y[first:first + 128], want, bound, str(first))
    del x, y
    buf = torch.zeros(2 ** 32 + 3 * 1024, dtype=BF16, device="cuda")
    rows = buf.as_strided((3, 512), (2 ** 31 + 8, 1))
    rows.copy_(_randn((3, 512), BF16, 1))
    _near(ops.dropout(rows, 0.25, _rng().cuda()), *ro.dropout(rows.cpu(), 0.25, ro.keep_mask(11, 5, 0.25, (3, 512))))


@pytest.mark.parametrize("with_residual", [False, True])
def test_dropout_where_the_counter_passes_32_bits(ops, with_residual):
    """Element 2^34 begins counter block 2^32."""
    n = 2 ** 34 + 100003
    x = torch.ones(n, dtype=BF16, device="cuda")
    y = ops.dropout(x, 0.25, _rng().cuda(), residual=x if with_residual else None)
    for first in (0, 2 ** 33, 2 ** 34 - 20000, 2 ** 34 - 64, 2 ** 34 + 64, n - 128):
        count = 40000 if first == 2 ** 34 - 20000 else 128
        keep = ro.keep_mask(11, 5, 0.25, (count,), first=first)
        one = torch.ones(count, dtype=BF16)
        want, bound = ro.dropout(one, 0.25, keep, one if with_residual else None)
        _near(y[first:first + count], want, bound, str(first))
    del x, y
    torch.cuda.empty_cache()


def test_generator_calls_and_replayed_graphs(ops):
    state = _rng(9, 0).cuda()
    taken = [ops.rng_take(state).tolist() for _ in range(3)]
    assert taken == [[9, 0], [9, 1], [9, 2]] and state.tolist() == [9, 3]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for i in range(20):
        with torch.cuda.stream(streams[i % 2]):
            got.append(ops.rng_take(state))
    torch.cuda.synchronize()
    assert sorted(g[1].item() for g in got) == list(range(3, 23))
    x = torch.ones(4, 64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.dropout(x, 0.5, ops.rng_take(state))
    for replay in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu() != 0, ro.keep_mask(9, 23 + replay, 0.5, (4, 64)))


def test_counter_dropout_module(ops):
    from hyc_lora_b200.operators.efficient_dropout import EfficientMemoryCounterDropout
    m = EfficientMemoryCounterDropout(0.3, seed=21, device="cuda")
    x = _randn((6, 40), F32, 1).cuda().requires_grad_(True)
    res = _randn((6, 40), F32, 2).cuda().requires_grad_(True)
    g = _randn((6, 40), F32, 3)
    for call in range(2):
        x.grad = res.grad = None
        y = m(x, res)
        y.backward(g.cuda())
        keep = ro.keep_mask(21, call, 0.3, (6, 40))
        _near(y, *ro.dropout(x.detach().cpu(), 0.3, keep, res.detach().cpu()))
        _near(x.grad, *ro.dropout(g, 0.3, keep))
        assert torch.equal(res.grad.cpu(), g)
    # a gradient that arrives expanded, and a mask handed in twice as a checkpointed function does
    rng = m.take()
    assert rng.tolist() == [21, 2]
    x.grad = None
    m(x, rng=rng).sum().backward()
    first = x.grad.clone()
    x.grad = None
    torch.utils.checkpoint.checkpoint(lambda t, r: m(t, rng=r), x, rng, use_reentrant=False).sum().backward()
    assert torch.equal(first, x.grad) and m.rng_state.tolist() == [21, 3]
    assert m.eval()(x) is x and m.rng_state.tolist() == [21, 3]


# ---------------------------------------------------------------------------------------------------- layer norm

NORM_COLS = [1, 2, 7, 8, 24, 100, 256, 257, 768, 1000, 1024, 1025, 2048, 4096, 4104, 5001, 8192, 11008, 16383, 16384]


def _norm_inputs(rows, cols, dtype, params, seed):
    x = _randn((rows, cols), dtype, seed, 2.0)
    if cols > 4:
        x[:, cols // 3] *= 30
    return x, (1 + _randn((cols,), F32, seed + 1, 0.2)).to(params), _randn((cols,), params, seed + 2, 0.2)


@pytest.mark.parametrize("cols", NORM_COLS)
@pytest.mark.parametrize("dtype,params", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("p,with_residual", [(0.0, False), (0.0, True), (0.25, False), (0.25, True)])
def test_layer_norm_matches_the_plain_form(ops, cols, dtype, params, p, with_residual):
    rows = 5 if cols > 2000 else 37
    x, w, b = _norm_inputs(rows, cols, dtype, params, cols)
    res = _randn((rows, cols), dtype, 9) if with_residual else None
    keep = ro.keep_mask(11, 5, p, x.shape)
    want, bounds = ro.layer_norm(x, w, b, 1e-5, res, p, keep)
    out = ops.layer_norm(x.cuda(), w.cuda(), b.cuda(), 1e-5, residual=None if res is None else res.cuda(), p=p, rng=_rng().cuda())
    for name, got, a, bound in zip(out._fields, out, want, bounds):
        _near(got, a, bound, name)
    # backward, from what the forward pass stored
    dy, extra = _randn((rows, cols), dtype, 7), _randn((rows, cols), dtype, 8) if with_residual else None
    got = ops.layer_norm_bwd(dy.cuda(), out.z, w.cuda(), out.mean, out.rstd, p=p, rng=_rng().cuda(),
                             dz=None if extra is None else extra.cuda())
    want, bounds = ro.layer_norm_bwd(dy, out.z.cpu(), w, out.mean.cpu(), out.rstd.cpu(), p, keep, extra, params)
    for name, a, v, bound in zip(("dx", "dresidual", "dweight", "dbias"), got, want, bounds):
        _near(a, v, bound, name)
    assert got[2].dtype == params and got[3].dtype == params


# Rows enough for every group of threads to take several: the forward pass with rows ahead in shared memory (from 4 rows per group
# and SM on: 4736, 1184 and 592 rows by the width), the sums of the parameter gradients over a group's rows, over groups and CTAs.
# Widths that fill their slots exactly (bounds are left out), that do not, and that are no multiple of eight.
MANY_ROWS = [(4740, 256), (4800, 248), (5000, 768), (5000, 760), (4800, 767), (5000, 1024), (4900, 1000), (1300, 2048), (1300, 1800),
             (1250, 2041), (1300, 4096), (1300, 4000), (700, 4095), (700, 6144), (700, 6000), (700, 8192), (700, 8184), (620, 8191),
             (700, 11008), (600, 12288), (600, 12287), (600, 16384), (600, 16000)]


@pytest.mark.parametrize("rows,cols", MANY_ROWS)
@pytest.mark.parametrize("dtype,params", [(BF16, F32), (F32, BF16)])
def test_layer_norm_of_many_rows(ops, rows, cols, dtype, params):
    x, w, b = _norm_inputs(rows, cols, dtype, params, cols)
    res, dy, dz = (_randn((rows, cols), dtype, s) for s in (9, 7, 8))
    keep = ro.keep_mask(11, 5, 0.2, x.shape)
    rng = _rng().cuda()
    out = ops.layer_norm(x.cuda(), w.cuda(), b.cuda(), 1e-5, residual=res.cuda(), p=0.2, rng=rng)
    for name, got, a, bound in zip(out._fields, out, *ro.layer_norm(x, w, b, 1e-5, res, 0.2, keep)):
        _near(got, a, bound, name)
    mean, rstd = out.mean.cpu(), out.rstd.cpu()
    got = ops.layer_norm_bwd(dy.cuda(), out.z, w.cuda(), out.mean, out.rstd, p=0.2, rng=rng, dz=dz.cuda())
    for name, a, v, bound in zip(("dx", "dresidual", "dweight", "dbias"), got, *ro.layer_norm_bwd(dy, out.z.cpu(), w, mean, rstd, 0.2, keep, dz, params)):
        _near(a, v, bound, name)
    # neither dropout nor a second gradient of the sum, no parameters
    out = ops.layer_norm(x.cuda(), None, None, 1e-5)
    for name, got, a, bound in zip(out._fields, out, *ro.layer_norm(x, None, None, 1e-5)):
        _near(got, a, bound, name)
    got = ops.layer_norm_bwd(dy.cuda(), out.z, None, out.mean, out.rstd, param_dtype=F32)
    for name, a, v, bound in zip(("dx", "dresidual", "dweight", "dbias"), got,
                                 *ro.layer_norm_bwd(dy, x, None, out.mean.cpu(), out.rstd.cpu(), param_dtype=F32)):
        _near(a, v, bound, name)


@pytest.mark.parametrize("rows", [0, 1, 2, 3, 31, 149, 1000, 5000])
@pytest.mark.parametrize("cols", [96, 99, 2056])
def test_layer_norm_row_counts(ops, rows, cols):
    x, w, b = _norm_inputs(rows, cols, BF16, F32, rows)
    keep = ro.keep_mask(11, 5, 0.1, x.shape)
    out = ops.layer_norm(x.cuda(), w.cuda(), b.cuda(), p=0.1, rng=_rng().cuda())
    want, bounds = ro.layer_norm(x, w, b, 1e-5, None, 0.1, keep)
    for got, a, bound in zip(out, want, bounds):
        _near(got, a, bound)
    dy = _randn((rows, cols), BF16, 7)
    got = ops.layer_norm_bwd(dy.cuda(), out.z, w.cuda(), out.mean, out.rstd, p=0.1, rng=_rng().cuda())
    want, bounds = ro.layer_norm_bwd(dy, out.z.cpu(), w, out.mean.cpu(), out.rstd.cpu(), 0.1, keep, None, F32)
    for a, v, bound in zip(got, want, bounds):
        _near(a, v, bound)
    again = ops.layer_norm_bwd(dy.cuda(), out.z, w.cuda(), out.mean, out.rstd, p=0.1, rng=_rng().cuda())
    assert all(torch.equal(a, v) for a, v in zip(got, again))       # the sums are taken in a fixed order


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cols", [64, 1024, 4096])
def test_layer_norm_of_unaligned_and_strided_rows(ops, dtype, cols):
    x, w, b = _norm_inputs(19, cols, dtype, dtype, 3)
    res, dy, dz = (_randn((19, cols), dtype, s) for s in (4, 5, 6))
    keep = ro.keep_mask(11, 5, 0.2, x.shape)
    want, bounds = ro.layer_norm(x, w, b, 1e-5, res, 0.2, keep)

    def spread(t, first, wide):
        buf = torch.full((19, cols + wide), 55.0, dtype=dtype, device="cuda")
        buf[:, first:first + cols] = t.cuda()
        return buf[:, first:first + cols]

    for first, wide in ((0, 8), (8, 16), (1, 8), (0, 5)):
        out = ops.layer_norm(spread(x, first, wide), _offset(w, first), _offset(b, first), residual=spread(res, first, wide), p=0.2, rng=_rng().cuda())
        for got, a, bound in zip(out, want, bounds):
            _near(got, a, bound, f"{first} {wide}")
        got = ops.layer_norm_bwd(spread(dy, first, wide), spread(out.z.cpu(), first, wide), _offset(w, first), out.mean, out.rstd, p=0.2,
                                 rng=_rng().cuda(), dz=spread(dz, first, wide))
        back, bb = ro.layer_norm_bwd(dy, out.z.cpu(), w, out.mean.cpu(), out.rstd.cpu(), 0.2, keep, dz, dtype)
        for a, v, bound in zip(got, back, bb):
            _near(a, v, bound, f"{first} {wide}")
    # an input that is expanded over its rows
    one = x[:1].expand(19, cols)
    out = ops.layer_norm(x[:1].cuda().expand(19, cols), w.cuda(), b.cuda())
    for got, a, bound in zip(out, *ro.layer_norm(one, w, b, 1e-5)):
        _near(got, a, bound, "expanded")


def test_layer_norm_beyond_32_bit_offsets(ops):
    buf = torch.zeros(2 ** 32 + 3 * 1024, dtype=BF16, device="cuda")
    x = buf.as_strided((3, 768), (2 ** 31 + 8, 1))
    x.copy_(_randn((3, 768), BF16, 1))
    out = ops.layer_norm(x, None, None)
    for got, a, bound in zip(out, *ro.layer_norm(x.cpu(), None, None, 1e-5)):
        _near(got, a, bound)
    dy = buf.as_strided((3, 768), (2 ** 31 + 8, 1), 1024)
    dy.copy_(_randn((3, 768), BF16, 2))
    got = ops.layer_norm_bwd(dy, x, None, out.mean, out.rstd)
    for a, v, bound in zip(got, *ro.layer_norm_bwd(dy.cpu(), x.cpu(), None, out.mean.cpu(), out.rstd.cpu())):
        _near(a, v, bound)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_layer_norm_without_parameters_or_variance(ops, dtype):
    x = torch.full((4, 96), 3.0, dtype=dtype)
    x[1] = 0.0
    x[2, 5] = 4.0
    b = _randn((96,), dtype, 1)
    for weight, bias in ((None, None), (None, b), (b, None)):
        out = ops.layer_norm(x.cuda(), None if weight is None else weight.cuda(), None if bias is None else bias.cuda())
        want, bounds = ro.layer_norm(x, weight, bias, 1e-5)
        for got, a, bound in zip(out, want, bounds):
            _near(got, a, bound)
        dy = _randn((4, 96), dtype, 2)
        for need_w, need_b in ((True, True), (True, False), (False, True), (False, False)):
            got = ops.layer_norm_bwd(dy.cuda(), out.z, None if weight is None else weight.cuda(), out.mean, out.rstd,
                                     need_dweight=need_w, need_dbias=need_b)
            back, bb = ro.layer_norm_bwd(dy, x, weight, out.mean.cpu(), out.rstd.cpu())
            assert (got[2] is not None) == need_w and (got[3] is not None) == need_b
            for a, v, bound in zip(got, back, bb):
                if a is not None:
                    _near(a, v, bound)


def test_layer_norm_row_with_nan_stays_its_own(ops):
    x, w, b = _norm_inputs(9, 768, BF16, BF16, 3)
    clean = ops.layer_norm(x.cuda(), w.cuda(), b.cuda())
    x[4, 100], x[6, 3] = float("nan"), INF
    out = ops.layer_norm(x.cuda(), w.cuda(), b.cuda())
    rows = torch.tensor([i for i in range(9) if i not in (4, 6)], device="cuda")
    assert torch.equal(out.y[rows], clean.y[rows]) and bool(out.y[4].isnan().all()) and bool(out.y[6].isnan().all())
    # what is dropped is not seen: the same places dropped leave no trace
    keep = ro.keep_mask(11, 5, 0.5, x.shape)
    x = torch.where(keep, _randn(x.shape, BF16, 5), torch.full_like(x, float("nan")))
    out = ops.layer_norm(x.cuda(), w.cuda(), b.cuda(), p=0.5, rng=_rng().cuda())
    for got, a, bound in zip(out, *ro.layer_norm(x, w, b, 1e-5, None, 0.5, keep)):
        _near(got, a, bound)


def test_layer_norm_far_from_zero_keeps_its_deviation(ops):
    """A mean a thousand deviations away: the deviation is taken about the mean, not from sums of squares."""
    x = (1000.0 + _randn((6, 768), F32, 1))
    out = ops.layer_norm(x.cuda(), None, None)
    for got, a, bound in zip(out, *ro.layer_norm(x, None, None, 1e-5)):
        _near(got, a, bound)


@pytest.mark.parametrize("return_sum", [False, True])
def test_norm_module_gradients_by_differences(ops, return_sum):
    """fp32, one direction at a time: the loss is a fixed weighting of the outputs, its derivative along a direction is taken
    from central differences.  The mask is fixed by handing ``rng`` in.  Truncation is h^2 times a third derivative (about
    1e-4 of the value here), rounding about 2^-24 * |loss terms| / h: h = 1e-2 leaves both under the 1e-3 allowed."""
    from hyc_lora_b200.operators.efficient_layernorm import EfficientMemoryDropoutAddLayerNorm
    m = EfficientMemoryDropoutAddLayerNorm(40, p=0.3, seed=3, return_sum=return_sum, device="cuda")
    with torch.no_grad():
        m.weight.copy_(1 + _randn((40,), F32, 1, 0.1))
        m.bias.copy_(_randn((40,), F32, 2, 0.1))
    x, res = (_randn((5, 40), F32, s).cuda().requires_grad_(True) for s in (3, 4))
    rng, a, b = m.take(), _randn((5, 40), F32, 5).cuda(), _randn((5, 40), F32, 6).cuda()

    def loss(x, res, w, bias):
        from hyc_lora_b200.operators.efficient_layernorm import DropoutAddLayerNormFunc
        y, z = DropoutAddLayerNormFunc.apply(x, res, w, bias, 1e-5, 0.3, rng)
        return (y.double() * a).sum() + ((z.double() * b).sum() if return_sum else 0.0)

    out = m(x, res, rng=rng)
    total = (out[0].double() * a).sum() + (out[1].double() * b).sum() if return_sum else (out.double() * a).sum()
    total.backward()
    at = [x.detach(), res.detach(), m.weight.detach(), m.bias.detach()]
    for i, grad in enumerate((x.grad, res.grad, m.weight.grad, m.bias.grad)):
        v = _randn(at[i].shape, F32, 20 + i).cuda()
        h = 1e-2
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + h * v, at[i] - h * v
        slope = (loss(*up) - loss(*down)).item() / (2 * h)
        scale = (grad.double().abs() * v.abs()).sum().item()
        assert abs(slope - (grad.double() * v).sum().item()) < 1e-3 * scale, i


def test_norm_module_paths(ops):
    from hyc_lora_b200.operators.efficient_layernorm import EfficientMemoryDropoutAddLayerNorm
    x, res = _randn((2, 3, 48), BF16, 1), _randn((2, 3, 48), BF16, 2)
    m = EfficientMemoryDropoutAddLayerNorm(48, p=0.4, seed=8, return_sum=True, device="cuda", dtype=BF16).eval()
    y, z = m(x.cuda(), res.cuda())                           # no dropout in evaluation
    (wy, wz, _, _), (by, bz, _, _) = ro.layer_norm(x, m.weight.cpu(), m.bias.cpu(), 1e-5, res)
    _near(y, wy, by)
    _near(z, wz, bz)
    assert m.rng_state.tolist() == [8, 0]
    xd = x.cuda().requires_grad_(True)
    y, z = m(xd)
    assert z is xd                                           # neither residual nor dropout: the sum is the input
    m.train()
    rd = res.cuda().requires_grad_(True)
    y, z = m(xd, rd)                                         # only the sum goes on
    z.sum().backward()
    keep = ro.keep_mask(8, 0, 0.4, x.shape)
    _near(xd.grad, *ro.dropout(torch.ones_like(x), 0.4, keep))
    assert bool((rd.grad == 1).all()) and m.weight.grad is None
    with pytest.raises(ValueError, match="residual has shape"):
        m(xd, rd[:1])
    with pytest.raises(TypeError):
        m(xd, rd.float())
    with pytest.raises(TypeError):
        m(xd.half())


# ---------------------------------------------------------------------------------------------------- token log probabilities

VOCABS = [1, 2, 7, 8, 33, 100, 256, 1000, 1001, 2048, 2049, 4097, 8200, 16384, 16385, 32000, 50265, 70001, 131072]


def _logit_inputs(rows, vocab, dtype, seed, masked=0.0):
    x = torch.randn((rows, vocab), generator=_gen(seed)) * 3
    t = torch.randint(0, vocab, (rows,), generator=_gen(seed + 1))
    x[torch.arange(rows), t] += torch.linspace(0, 40, rows)     # from unlikely to certain
    if masked:
        shut = torch.rand((rows, vocab), generator=_gen(seed + 2)) < masked
        shut[torch.arange(rows), t] = False
        how = torch.where(torch.rand((rows, vocab), generator=_gen(seed + 3)) < 0.5, -INF, torch.finfo(dtype).min)
        x = torch.where(shut, how, x)
    return x.to(dtype), t


def _check_logprobs(ops, x, t, xd, top, entropy=True, ignore=-100):
    out = ops.token_logprobs(xd, None if t is None else t.cuda(), entropy=entropy, top=top, ignore_index=ignore)
    want, bound = ro.token_logprobs(x, t, ignore, top)
    if t is not None:
        _near(out.logprob, want["logprob"], bound["logprob"], "logprob")
    if entropy:
        _near(out.entropy, want["entropy"], bound["entropy"], "entropy")
    if top:
        assert torch.equal(out.top_index.cpu(), want["top_index"])
        _near(out.top_logprob, want["top_logprob"], bound["top_logprob"], "alternatives")
    _near(out.stats, want["stats"], bound["stats"], "stats")
    return out


def _check_grads(ops, x, xd, out, t, top, ignore=-100):
    rows = x.shape[0]
    d1, d2 = _randn((rows,), F32, 50), _randn((rows,), F32, 51)
    d3 = _randn((rows, top), F32, 52) if top else None
    stats, h = out.stats.cpu(), out.entropy.cpu()
    index = out.top_index if top else None
    for use in ((1, 0, 0), (0, 1, 0), (1, 1, 0), (1, 1, 1), (0, 0, 1)):
        if use[2] and not top:
            continue
        got = ops.token_logprobs_bwd(xd, out.stats, t.cuda() if use[0] else None, d1.cuda() if use[0] else None, ignore_index=ignore,
                                     entropy=out.entropy if use[1] else None, d_entropy=d2.cuda() if use[1] else None,
                                     top_index=index if use[2] else None, d_top=d3.cuda() if use[2] else None)
        want, bound = ro.token_logprobs_bwd(x, stats, t, d1 if use[0] else None, ignore, h if use[1] else None, d2 if use[1] else None,
                                            index.cpu() if use[2] else None, d3 if use[2] else None)
        assert got.dtype == x.dtype
        _near(got, want, bound, f"gradient {use}")


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logprobs_match_the_plain_form(ops, vocab, dtype):
    rows = 9 if vocab < 20000 else 5
    x, t = _logit_inputs(rows, vocab, dtype, vocab)
    t[rows // 2] = -100
    for top in sorted({0, 1, min(5, vocab), min(32, vocab)}):
        out = _check_logprobs(ops, x, t, x.cuda(), top)
    _check_grads(ops, x, x.cuda(), out, t, min(32, vocab))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logprobs_at_the_largest_vocabulary(ops, dtype):
    x, t = _logit_inputs(3, 262144, dtype, 5)
    out = _check_logprobs(ops, x, t, x.cuda(), 20)
    _check_grads(ops, x, x.cuda(), out, t, 20)
    with pytest.raises(RuntimeError, match="exceeds"):
        ops.token_logprobs(torch.zeros(1, 262145, dtype=dtype, device="cuda"))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab,masked", [(40, 0.5), (1003, 0.3), (32000, 0.9), (32000, 0.9995), (70001, 0.99999)])
def test_logprobs_of_masked_vocabularies(ops, dtype, vocab, masked):
    x, t = _logit_inputs(6, vocab, dtype, 31, masked)
    for top in (0, 1, 20):
        out = _check_logprobs(ops, x, t, x.cuda(), top)
    _check_grads(ops, x, x.cuda(), out, t, 20)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [5, 1000, 32000, 50265])
def test_logprobs_of_rows_without_a_choice(ops, dtype, vocab):
    """No open token; one open token; all equal; all at the type's lowest value; two equal best ones."""
    low = torch.finfo(dtype).min
    x = torch.full((7, vocab), -INF, dtype=dtype)
    x[1, vocab // 2] = 3.0
    x[2] = 1.5
    x[3] = low
    x[4] = _randn((vocab,), dtype, 1)
    x[4, [1, vocab - 1]] = 20.0
    x[5] = low
    x[5, 2] = -INF
    x[6] = 0.0
    x[6, ::2] = -0.0                                          # zeros of both signs are equal
    t = torch.tensor([0, vocab // 2, vocab - 1, 2, vocab - 1, 1, 3])
    for top in (0, 1, 4):
        out = _check_logprobs(ops, x, t, x.cuda(), top)
    assert out.logprob[0].item() == -INF and out.entropy[0].item() == 0.0 and out.stats[0].tolist() == [-INF, 0.0]
    assert out.top_index[0].tolist() == [0, 1, 2, 3] and out.top_index[6].tolist() == [0, 1, 2, 3]
    _check_grads(ops, x, x.cuda(), out, t, 4)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,vocab", [(5, 700), (3, 32000), (300, 4100), (3, 100003)])
def test_logprobs_alternatives_among_very_many_equal_values(ops, dtype, rows, vocab):
    """Rows whose k-th best value is shared by more elements than are collected: a few open tokens among masked ones, two levels,
    equal values that begin late in the row."""
    low = torch.finfo(dtype).min
    x = torch.full((rows, vocab), -INF, dtype=dtype)
    x[0, [vocab - 1, 3, vocab // 2]] = torch.tensor([1.0, 5.0, 5.0], dtype=dtype)
    x[1] = low
    x[1, vocab // 3:vocab // 3 + 7] = _randn((7,), dtype, 1)
    x[2, : vocab // 2] = -3.0
    x[2, vocab // 2:] = 2.0
    x[2, -1] = 4.0
    for row in range(3, rows):
        x[row] = low if row % 2 else -INF
        open_ = torch.randperm(vocab, generator=_gen(row))[: row % 25]
        x[row, open_] = _randn((len(open_),), dtype, row)
    t = torch.arange(rows) % vocab
    for top in (1, 4, 20, 32):
        _check_logprobs(ops, x, t, x.cuda(), top)
    _check_logprobs(ops, x, t, _offset(x, 1), 20)


@pytest.mark.parametrize("vocab", [300, 3001, 40000, 100001])
def test_logprobs_with_nan_and_infinity(ops, vocab):
    """Short rows, rows of one CTA and rows that are spread over a cluster, of which one slice holds the NaN."""
    x, t = _logit_inputs(5, vocab, F32, 3)
    t[1] = 7
    x[1, vocab // 3], x[2, 5] = float("nan"), INF
    out = ops.token_logprobs(x.cuda(), t.cuda(), entropy=True, top=3)
    for row in (1, 2):
        assert out.logprob[row].isnan() and out.entropy[row].isnan() and bool(out.top_logprob[row].isnan().all())
    assert out.top_index[1, 0].item() == vocab // 3 and out.top_index[2, 0].item() == 5
    finite = x[1].clone()
    finite[vocab // 3] = -INF
    assert out.top_index[1, 1].item() == finite.argmax().item()
    rest = torch.tensor([0, 3, 4])
    want, bound = ro.token_logprobs(x[rest], t[rest], top=3)
    _near(out.logprob[rest.cuda()], want["logprob"], bound["logprob"])
    assert torch.equal(out.top_index[rest.cuda()].cpu(), want["top_index"])
    g = ops.token_logprobs_bwd(x.cuda(), out.stats, t.cuda(), torch.ones(5, device="cuda"))
    assert bool(g[1].isnan().all()) and bool(g[2].isnan().all()) and not bool(g[rest.cuda()].isnan().any())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [1, 4, 20, 32, 300, 3001, 40000, 100001])
@pytest.mark.parametrize("where", ["first", "all", "ends", "both signs"])
def test_logprobs_nan_is_an_alternative_wherever_it_stands(ops, dtype, vocab, where):
    """A NaN stands above +inf, the lower index first among several; every index lies in the vocabulary, also where all of it
    is asked for."""
    x, t = _logit_inputs(4, vocab, dtype, 3)
    if where == "first":
        x[:, 0] = float("nan")
    elif where == "all":
        x[:] = float("nan")
    elif where == "ends":
        x[:, vocab - 1] = float("nan")
        x[1, 0] = float("nan")
        x[2, vocab // 2] = INF
    else:
        x[:, 0] = -torch.tensor(float("nan"))
        x[:, vocab // 2] = float("nan")
    x[3] = _randn((vocab,), dtype, 5)                         # a row without
    rank = torch.where(x.isnan(), torch.full_like(x, INF, dtype=torch.float64), x.double().clamp_max(1e300))
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices
    for top in sorted({1, min(5, vocab), min(32, vocab)}):
        out = ops.token_logprobs(x.cuda(), t.cuda(), entropy=True, top=top)
        assert torch.equal(out.top_index.cpu(), order[:, :top]), top
        assert bool(out.top_logprob[:3].isnan().all()) and not bool(out.top_logprob[3].isnan().any())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shift", [1000.0, -30000.0, 1.04e6, -1.2e6, 3e9, 1e20, -1e29, 1e31, -1e36])
@pytest.mark.parametrize("rows,vocab", [(6, 1000), (6, 33000), (700, 2100)])
def test_logprobs_of_logits_far_from_zero(ops, dtype, shift, rows, vocab):
    """The differences are what counts: neither the size of the logits nor their sign costs digits."""
    x, t = _logit_inputs(rows, vocab, F32, 9)
    x = (x + shift).to(dtype)
    out = _check_logprobs(ops, x, t, x.cuda(), 5)
    if rows < 100:
        _check_grads(ops, x, x.cuda(), out, t, 5)


def test_logprobs_targets_outside_and_ignored(ops):
    x, t = _logit_inputs(6, 1000, BF16, 3)
    t[0], t[1], t[2], t[3] = -100, 1000, -1, 2 ** 40
    for extra in (dict(), dict(entropy=True)):
        out = ops.token_logprobs(x.cuda(), t.cuda(), **extra)
        assert out.logprob[0].item() == 0.0 and bool(out.logprob[1:4].isnan().all()) and not bool(out.logprob[4:].isnan().any())
    d = torch.ones(6, device="cuda")
    g = ops.token_logprobs_bwd(x.cuda(), out.stats, t.cuda(), d)
    assert bool((g[0] == 0).all()) and bool(g[1:4].isnan().all()) and not bool(g[4:].isnan().any())
    # an ignored row that nothing else is asked of is not read: what it holds does not matter
    skipped = ops.token_logprobs(torch.where(torch.arange(6)[:, None] == 0, float("nan"), x.float()).to(BF16).cuda(), t.cuda())
    assert skipped.logprob[0].item() == 0.0 and skipped.stats[0].tolist() == [-INF, 0.0]
    g = ops.token_logprobs_bwd(x.cuda(), skipped.stats, t.cuda(), d)
    assert bool((g[0] == 0).all())
    # another ignore_index, which may be a token of the vocabulary
    t = torch.tensor([3, 4, 3, 5, 6, 3])
    _check_logprobs(ops, x, t, x.cuda(), 2, ignore=3)
    assert ops.token_logprobs(x.cuda(), entropy=True).logprob is None


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("vocab", [65, 1000, 32000])
def test_logprobs_of_unaligned_and_strided_logits(ops, dtype, vocab):
    x, t = _logit_inputs(12, vocab, dtype, 3)
    for off in (1, 3, 4):
        out = _check_logprobs(ops, x, t, _offset(x, off), 3)
        _check_grads(ops, x, _offset(x, off), out, t, 3)
    # the shifted view of a batch: two leading strides
    batch = x.view(3, 4, vocab).cuda()
    view, flat = batch[:, :-1], x.view(3, 4, vocab)[:, :-1].reshape(9, vocab)
    tt = t.view(3, 4)[:, 1:].contiguous()
    out = ops.token_logprobs(view, tt.cuda(), entropy=True, top=2)
    want, bound = ro.token_logprobs(flat, tt.reshape(-1), top=2)
    _near(out.logprob.reshape(-1), want["logprob"], bound["logprob"])
    assert out.logprob.shape == (3, 3) and out.top_index.shape == (3, 3, 2)
    assert torch.equal(out.top_index.reshape(9, 2).cpu(), want["top_index"])
    d = _randn((3, 3), F32, 1)
    got = ops.token_logprobs_bwd(view, out.stats, tt.cuda(), d.cuda())
    back, bb = ro.token_logprobs_bwd(flat, out.stats.cpu(), tt.reshape(-1), d.reshape(-1))
    assert got.shape == view.shape and got.is_contiguous()
    _near(got.reshape(9, vocab), back, bb)
    # a column slice, and columns that lie apart (copied)
    wide = torch.cat((x, x), 1).cuda()
    _check_logprobs(ops, x, t, wide[:, :vocab], 1)
    _check_logprobs(ops, x, t, wide[:, vocab:], 1)
    _check_logprobs(ops, x, t, x.t().contiguous().cuda().t(), 1)


def test_logprobs_beyond_32_bit_offsets(ops):
    vocab = 32000
    buf = torch.zeros(2 ** 32 + vocab + 64, dtype=BF16, device="cuda")
    xd = buf.as_strided((3, vocab), (2 ** 31 + 24, 1))
    x, t = _logit_inputs(3, vocab, BF16, 3)
    xd.copy_(x)
    out = _check_logprobs(ops, x, t, xd, 3)
    del buf
    rows = 140000                                             # a gradient of more than 2^32 elements
    big = torch.zeros((rows, vocab), dtype=BF16, device="cuda")
    big[-3:] = x.cuda()
    stats = torch.zeros((rows, 2), device="cuda")
    stats[:, 0] = -INF
    stats[-3:] = out.stats
    tt = torch.zeros(rows, dtype=torch.int64, device="cuda")
    tt[-3:] = t.cuda()
    g = ops.token_logprobs_bwd(big, stats, tt, torch.ones(rows, device="cuda"))
    _near(g[-3:], *ro.token_logprobs_bwd(x, out.stats.cpu(), t, torch.ones(3)))
    assert int(torch.count_nonzero(g[:-3])) == 0
    # three rows are spread over clusters, 140000 are not: the sums run in another order, each within the counted roundings
    again = ops.token_logprobs(big, tt)
    want, bound = ro.token_logprobs(x, t)
    _near(again.stats[-3:], want["stats"], bound["stats"])
    _near(again.logprob[-3:], want["logprob"], bound["logprob"])


def test_logprobs_of_no_rows_and_of_one_vector(ops):
    out = ops.token_logprobs(torch.empty(0, 100, dtype=BF16, device="cuda"), torch.empty(0, dtype=torch.int64, device="cuda"), entropy=True, top=2)
    assert out.logprob.shape == (0,) and out.top_index.shape == (0, 2)
    assert ops.token_logprobs_bwd(torch.empty(0, 100, device="cuda"), out.stats).shape == (0, 100)
    x, _ = _logit_inputs(1, 100, F32, 1)
    one = ops.token_logprobs(x[0].cuda(), torch.tensor(3).cuda(), top=2)
    assert one.logprob.shape == () and one.top_index.shape == (2,)
    for bad in (dict(top=101), dict(top=33), dict(top=-1)):
        with pytest.raises(RuntimeError):
            ops.token_logprobs(x.cuda(), **bad)
    with pytest.raises(TypeError):
        ops.token_logprobs(x.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        ops.token_logprobs(x.cuda(), torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(TypeError):
        ops.token_logprobs(x.cuda().half())


@pytest.mark.parametrize("rows,vocab", [(1, 32000), (2, 2000), (150, 129), (700, 2000), (1500, 300), (5000, 40), (313, 8200), (600, 16500)])
def test_logprobs_row_counts(ops, rows, vocab):
    x, t = _logit_inputs(rows, vocab, BF16, rows)
    t[::3] = -100
    for top in (0, 3):
        out = _check_logprobs(ops, x, t, x.cuda(), top)
    plain = ops.token_logprobs(x.cuda(), t.cuda())
    want, bound = ro.token_logprobs(x, t)
    _near(plain.logprob, want["logprob"], bound["logprob"], "targets alone")
    d = _randn((rows,), F32, 1)
    _near(ops.token_logprobs_bwd(x.cuda(), plain.stats, t.cuda(), d.cuda()), *ro.token_logprobs_bwd(x, out.stats.cpu(), t, d))


@pytest.mark.parametrize("rows,vocab", [(1, 262144), (2, 32000), (40, 16385), (96, 70001), (130, 33000)])
def test_logprobs_of_clusters_that_find_little_to_do(ops, rows, vocab):
    """Rows spread over CTAs that meet at their start: all of them ignored (nothing is read), every other one, only the last."""
    x, t = _logit_inputs(rows, vocab, BF16, rows)
    xd = x.cuda()
    for ignored in (torch.ones(rows, dtype=torch.bool), torch.arange(rows) % 2 == 0, torch.arange(rows) < rows - 1):
        tt = torch.where(ignored, -100, t)
        got = ops.token_logprobs(xd, tt.cuda())
        want, bound = ro.token_logprobs(x, tt)
        _near(got.logprob, want["logprob"], bound["logprob"])
        assert bool((got.stats.cpu()[ignored] == torch.tensor([-INF, 0.0])).all())
        _near(got.stats[~ignored.cuda()], want["stats"][~ignored], bound["stats"][~ignored])
        again = ops.token_logprobs(xd, tt.cuda(), entropy=True, top=7)
        want, bound = ro.token_logprobs(x, tt, top=7)
        assert torch.equal(again.top_index.cpu(), want["top_index"])
        _near(again.entropy, want["entropy"], bound["entropy"])


def test_logprob_gradient_with_repeated_and_foreign_alternatives(ops):
    """An index that repeats, equals the target, or lies outside the vocabulary (which takes part in the sum only)."""
    x, t = _logit_inputs(4, 500, F32, 3)
    out = ops.token_logprobs(x.cuda())
    index = torch.tensor([[5, 5, 9, 5]] * 4)
    index[:, 2] = t
    d, dt = _randn((4, 4), F32, 1), _randn((4,), F32, 2)
    args = (x.cuda(), out.stats, t.cuda(), dt.cuda())
    _near(ops.token_logprobs_bwd(*args, top_index=index.cuda(), d_top=d.cuda()),
          *ro.token_logprobs_bwd(x, out.stats.cpu(), t, dt, top_index=index, d_top=d))
    foreign = index.clone()
    foreign[:, 0], foreign[:, 3] = -1, 500
    got = ops.token_logprobs_bwd(*args, top_index=foreign.cuda(), d_top=d.cuda())
    p = ro.token_logprobs(x, t)[0]
    lost = d[:, [0, 3]].double().sum(1, keepdim=True) * (x.double() - p["stats"].sum(1, keepdim=True)).exp()
    want, bound = ro.token_logprobs_bwd(x, out.stats.cpu(), t, dt, top_index=index[:, 1:3], d_top=d[:, 1:3])
    _near(got, want - lost, bound + lost.abs() * 200 * ro.U)


def test_logprob_function_by_autograd(ops):
    from hyc_lora_b200.operators.efficient_logprob import EfficientMemoryTokenLogprob, token_cross_entropy
    x, t = _logit_inputs(8, 300, F32, 5)
    t[3] = -100
    d1, d2, d3 = _randn((8,), F32, 1), _randn((8,), F32, 2), _randn((8, 4), F32, 3)
    xd = x.cuda().requires_grad_(True)
    logprob, entropy, best, index = EfficientMemoryTokenLogprob(entropy=True, top=4)(xd, t.cuda())
    assert not index.requires_grad
    ((logprob * d1.cuda()).sum() + (entropy * d2.cuda()).sum() + (best * d3.cuda()).sum()).backward()
    ref = x.double().requires_grad_(True)
    lp = torch.log_softmax(ref, 1)
    total = (torch.where(t == -100, 0.0, lp.gather(1, t.clamp_min(0)[:, None])[:, 0]) * d1).sum()
    total = total - ((lp.exp() * lp).sum(1) * d2).sum() + (lp.topk(4, 1).values * d3).sum()
    total.backward()
    want, bound = ro.token_logprobs_bwd(x, ops.token_logprobs(x.cuda()).stats.cpu(), t, d1, entropy=entropy.detach().cpu(), d_entropy=d2,
                                        top_index=index.cpu(), d_top=d3)
    assert (want - ref.grad).abs().max() < 1e-5              # the formula from the stored fp32 statistics against autograd in 64 bits
    _near(xd.grad, want, bound)
    # differences: the same direction in both, h^2 truncation (third derivative of order 1) and 2^-24 / h rounding under 2e-3
    v = _randn(x.shape, F32, 9).cuda()

    def loss(z):
        a, b, c, _ = EfficientMemoryTokenLogprob(entropy=True, top=4)(z, t.cuda())
        return ((a.double() * d1.cuda()).sum() + (b.double() * d2.cuda()).sum() + (c.double() * d3.cuda()).sum()).item()

    h = 3e-3
    slope = (loss(x.cuda() + h * v) - loss(x.cuda() - h * v)) / (2 * h)
    assert abs(slope - (xd.grad.double() * v).sum().item()) < 2e-3 * (xd.grad.double() * v).abs().sum().item()
    # the loss made of it
    for reduction in ("mean", "sum", "none"):
        a, b = x.cuda().requires_grad_(True), x.double().requires_grad_(True)
        la = token_cross_entropy(a, t.cuda(), reduction=reduction)
        lb = torch.nn.functional.cross_entropy(b, t, reduction=reduction)
        la.sum().backward()
        lb.sum().backward()
        assert (la.detach().cpu().double() - lb.detach()).abs().max() < 1e-4 and (a.grad.cpu().double() - b.grad).abs().max() < 1e-6
    assert token_cross_entropy(x.cuda(), torch.full((8,), -100, device="cuda")).isnan()
    only_index = EfficientMemoryTokenLogprob(top=2)(x.cuda())
    assert only_index[0] is None and only_index[3].shape == (8, 2)


# ---------------------------------------------------------------------------------------------------- together

def test_operators_on_another_stream_and_in_two_graphs(ops):
    """Two graphs recorded one after the other and replayed in turn on streams of their own share nothing."""
    rows, cols, vocab = 300, 776, 4000
    w, b = _randn((cols,), BF16, 1).cuda(), _randn((cols,), BF16, 2).cuda()
    state = _rng(3, 0).cuda()

    def step(x, logits, t, rng):
        out = ops.layer_norm(x, w, b, residual=x, p=0.2, rng=rng)
        back = ops.layer_norm_bwd(x, out.z, w, out.mean, out.rstd, p=0.2, rng=rng)
        lp = ops.token_logprobs(logits, t, entropy=True, top=3)
        return [*out, *back, lp.logprob, lp.entropy, lp.top_index, ops.token_logprobs_bwd(logits, lp.stats, t, lp.logprob)]

    rng = ops.rng_take(state)
    data = []
    for s in (5, 6):
        x, t = _logit_inputs(rows, vocab, BF16, s)
        data.append((_randn((rows, cols), BF16, s).cuda(), x.cuda(), t.cuda(), rng))
    want = [step(*d) for d in data]
    graphs, outs = [], []
    for d in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*d))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, a in zip(outs, want):
        assert all(torch.equal(p, q) for p, q in zip(o, a))
    with torch.cuda.stream(streams[0]):
        got = step(*data[1])
    streams[0].synchronize()
    assert all(torch.equal(p, q) for p, q in zip(got, want[1]))


def test_decoder_host_with_the_fused_loss(ops):
    from hyc_lora_b200 import synthetic
    from hyc_lora_b200.hosts.llama import DecoderConfig, DecoderLM
    cfg = DecoderConfig(hidden=512, layers=2, heads=4, kv_heads=2, ffn=1408, vocab=1001, lora_r=16, base_quant="nf4")
    model = DecoderLM(cfg, seed=1)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for n, q in model.named_parameters():
        if "lora_B" in n:
            q.data.normal_(0, 0.05, generator=gen)
    ids = synthetic.token_ids(3, 2, 64, cfg.vocab).cuda()
    model(ids).backward()
    want = {n: q.grad.clone() for n, q in model.named_parameters() if q.grad is not None}
    fused = copy.deepcopy(model)
    fused.zero_grad(set_to_none=True)
    fused.config.fused_loss = True
    loss = fused(ids)
    loss.backward()
    fused.config.fused_loss = False
    with torch.no_grad():
        # the same logits: fp32 sums of 63 * 2 terms of about 7, each within a few 2^-24
        assert abs(loss.item() - fused(ids).item()) < 1e-4
    for n, q in fused.named_parameters():
        if q.grad is not None:
            # both hand bf16 gradients of the logits on, rounded once from fp32: they differ by a rounding here and there
            cos = torch.nn.functional.cosine_similarity(q.grad.float().flatten(), want[n].float().flatten(), dim=0)
            assert cos > 0.999, (n, cos.item())
    got = model.score(ids, entropy=True, top=3)
    logits = model.logits(ids).detach().cpu()
    nxt = torch.nn.functional.pad(ids[:, 1:], (0, 1), value=-100).cpu()
    ref, bound = ro.token_logprobs(logits.reshape(-1, cfg.vocab), nxt.reshape(-1), top=3)
    _near(got.logprob.reshape(-1), ref["logprob"], bound["logprob"])
    _near(got.entropy.reshape(-1), ref["entropy"], bound["entropy"])
    assert torch.equal(got.top_index.reshape(-1, 3).cpu(), ref["top_index"])


def test_fused_loss_hands_the_same_gradient_to_the_logits(ops):
    """Both losses give the logits' gradient in bf16, rounded once from fp32: two values that are each within half a step of the
    formula's are at most one step (2^-7 of the value) apart; 2^-20 of it is for the fp32 arithmetic, softmax and quotient."""
    from hyc_lora_b200 import synthetic
    from hyc_lora_b200.hosts.llama import DecoderConfig, DecoderLM
    cfg = DecoderConfig(hidden=512, layers=1, heads=4, kv_heads=2, ffn=1408, vocab=1001, lora_r=16, base_quant="nf4")
    model = DecoderLM(cfg, seed=1)
    ids = synthetic.token_ids(3, 3, 33, cfg.vocab).cuda()
    kept = []
    model.lm_head.register_forward_hook(lambda module, args, out: (out.retain_grad(), kept.append(out))[0])
    grads = []
    for fused in (False, True):
        model.zero_grad(set_to_none=True)
        model.config.fused_loss = fused
        model(ids).backward()
        grads.append({n for n, q in model.named_parameters() if q.grad is not None})
    assert grads[0] == grads[1] and len(grads[0]) > 0
    plain, fused = kept
    assert torch.equal(plain, fused) and plain.grad.dtype == fused.grad.dtype == BF16
    a, b = plain.grad.double(), fused.grad.double()
    assert bool((b[:, -1] == 0).all()) and bool(((a - b).abs() <= (2.0 ** -7 + 2.0 ** -20) * torch.minimum(a.abs(), b.abs())).all())
    x, t = plain.detach().double()[:, :-1], ids[:, 1:]
    want = (torch.softmax(x, -1) - torch.nn.functional.one_hot(t, cfg.vocab)) / t.numel()
    assert bool(((b[:, :-1] - want).abs() <= (2.0 ** -8 + 2.0 ** -18) * want.abs()).all())


@pytest.mark.parametrize("mode", ["element", "channel"])
@pytest.mark.parametrize("scored_before", [0, 1, 2, 3])
def test_scoring_leaves_the_calibration_alone(ops, mode, scored_before):
    """A model with compression operators that is scored on other text before its training step ``scored_before``, and a copy that
    is not: the same calibration and, to the bit, the same losses and gradients."""
    from hyc_lora_b200 import synthetic
    from hyc_lora_b200.hosts.llama import DecoderConfig, DecoderLM
    from hyc_lora_b200.hosts.replace import replace_module, uniform_config
    from hyc_lora_b200.operators._common import calibration_state_dict
    cfg = DecoderConfig(hidden=512, layers=2, heads=4, kv_heads=2, ffn=1408, vocab=1001, lora_r=16, base_quant="nf4", fused_loss=True)
    model = DecoderLM(cfg, seed=1)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for n, q in model.named_parameters():
        if "lora_B" in n:
            q.data.normal_(0, 0.05, generator=gen)
    extra = dict(outlier_mode="channel", rotate=64) if mode == "channel" else {}
    assert replace_module(model, uniform_config(outlier_ratio=0.02), extra) > 0
    other = copy.deepcopy(model)
    for step in range(5):
        ids = synthetic.token_ids(10 + step, 2, 64, cfg.vocab).cuda()
        results = []
        for m in (model, other):
            if m is model and step >= scored_before:
                text = synthetic.token_ids(90 + step, 3, 40, cfg.vocab).cuda()
                got = m.score(text, entropy=True, top=2)
                assert torch.equal(got.logprob, m.score(text).logprob)
            m.zero_grad(set_to_none=True)
            loss = m(ids)
            loss.backward()
            results.append((loss.item(), {n: q.grad for n, q in m.named_parameters() if q.grad is not None}))
        (a, ga), (b, gb) = results
        assert a == b and ga.keys() == gb.keys() and len(ga) > 0
        assert all(torch.equal(ga[n], gb[n]) for n in ga), step
    for (n, p), (_, q) in zip(model.named_modules(), other.named_modules()):
        if hasattr(p, "iteration"):
            assert p.iteration == 5 and _same(calibration_state_dict(p), calibration_state_dict(q)), n


@pytest.mark.parametrize("mode", ["none", "element", "channel"])
def test_scoring_in_inference_mode(ops, mode):
    """The very first call of a model in inference mode, then outside, then a training step: nothing made in the one is kept for
    the others."""
    from hyc_lora_b200 import synthetic
    from hyc_lora_b200.hosts.llama import DecoderConfig, DecoderLM
    from hyc_lora_b200.hosts.replace import replace_module, uniform_config
    cfg = DecoderConfig(hidden=256, layers=2, heads=4, kv_heads=2, ffn=512, vocab=301, lora_r=16, rope_theta=9000.0, fused_loss=True)
    model = DecoderLM(cfg, seed=1)
    if mode != "none":
        replace_module(model, uniform_config(outlier_ratio=0.02), dict(outlier_mode="channel", rotate=64) if mode == "channel" else {})
    ids = synthetic.token_ids(3, 2, 48, cfg.vocab).cuda()
    with torch.inference_mode():
        got = model.score(ids.clone(), entropy=True, top=3)
    want = model.score(ids, entropy=True, top=3)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for _ in range(3):
        model(ids).backward()
    assert all(bool(q.grad.isfinite().all()) for q in model.parameters() if q.requires_grad)


def _same(a, b):
    if torch.is_tensor(a):
        return torch.is_tensor(b) and torch.equal(a, b)
    if isinstance(a, dict):
        return a.keys() == b.keys() and all(_same(a[k], b[k]) for k in a)
    if isinstance(a, (list, tuple)):
        return len(a) == len(b) and all(_same(p, q) for p, q in zip(a, b))
    return a == b


def test_encoder_host_with_hidden_dropout(ops):
    """The whole host with its dropouts against the same host with the masks applied by tensor ops, and a recorded step."""
    from hyc_lora_b200.hosts.roberta import EncoderClassifier, EncoderConfig
    cfg = EncoderConfig(hidden=128, layers=2, heads=4, ffn=256, vocab=200, max_pos=66, lora_r=8, hidden_dropout=0.2)
    torch.manual_seed(4)
    model = EncoderClassifier(cfg, seed=2)
    for layer in model.layers:
        layer.attention.dropout.p = 0.0                       # torch's own generator stays out of the comparison
    model.train()
    ids = torch.randint(0, 200, (3, 32), generator=_gen(1)).cuda()
    labels = torch.tensor([0, 1, 1]).cuda()
    states = [m.rng_state.tolist() for m in model.modules() if hasattr(m, "rng_state")]
    assert len(states) == 5 and len({s[0] for s in states}) == 5
    loss = model(ids, labels)
    loss.backward()
    grads = {n: q.grad.clone() for n, q in model.named_parameters() if q.grad is not None}
    calls = {id(m): m.rng_state.tolist() for m in model.modules() if hasattr(m, "rng_state")}

    def masked(module, x):
        seed, call = calls[id(module)]
        keep = ro.keep_mask(seed, call - 1, 0.2, x.shape).cuda()
        return torch.where(keep, x / 0.8, torch.zeros_like(x))

    for layer in model.layers:
        for norm in (layer.attn_LayerNorm, layer.out_LayerNorm):
            norm.forward = lambda x, residual, n=norm: torch.nn.functional.layer_norm(masked(n, x) + residual, (128,), n.weight, n.bias, n.eps)
    model.emb_dropout.forward = lambda x, d=model.emb_dropout: masked(d, x)
    model.zero_grad(set_to_none=True)
    want = model(ids, labels)
    want.backward()
    assert abs(want.item() - loss.item()) < 1e-4
    for n, q in model.named_parameters():
        if q.grad is not None:
            # fp32 throughout, sums of a few hundred terms in another order
            assert (q.grad - grads[n]).abs().max() <= 1e-3 * grads[n].abs().max() + 1e-6, n


def test_encoder_step_replays_with_new_masks(ops):
    from hyc_lora_b200.hosts.roberta import EncoderClassifier, EncoderConfig
    from hyc_lora_b200.hosts.step import Trainer
    torch.manual_seed(4)
    model = EncoderClassifier(EncoderConfig(hidden=128, layers=1, heads=4, ffn=256, vocab=200, max_pos=66, lora_r=8, hidden_dropout=0.2), seed=2)
    model.layers[0].attention.dropout.p = 0.0
    model.train()
    labels = torch.tensor([0, 1, 1]).cuda()
    ids = torch.randint(0, 200, (3, 32), generator=_gen(1)).cuda()
    trainer = Trainer(_WithLabels(model, labels), lr=0.0)
    assert trainer.capture(ids)
    before = model.emb_dropout.rng_state[1].item()
    losses = {round(trainer.step(ids).item(), 7) for _ in range(4)}
    assert model.emb_dropout.rng_state[1].item() == before + 4
    assert len(losses) > 1                                    # nothing moves but the masks


class _WithLabels(torch.nn.Module):
    def __init__(self, model, labels):
        super().__init__()
        self.model, self.labels = model, labels

    def forward(self, ids):
        return self.model(ids, self.labels)


def test_first_calls_inside_a_capture():
    """A fresh process whose very first call of each operator is recorded into a graph."""
    import subprocess
    import sys
    code = """
import torch
from hyc_lora_b200 import rowops as o
x = torch.randn(2500, 4096, device='cuda', dtype=torch.bfloat16)
w, lg, t = torch.ones(4096, device='cuda'), torch.randn(8, 70000, device='cuda'), torch.zeros(8, dtype=torch.int64, device='cuda')
state = torch.tensor([1, 0], device='cuda')
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    rng = o.rng_take(state)
    out = o.layer_norm(o.dropout(x, 0.1, rng, residual=x), w, w, residual=x, p=0.1, rng=rng)
    back = o.layer_norm_bwd(x, out.z, w, out.mean, out.rstd, p=0.1, rng=rng)
    lp = o.token_logprobs(lg, t, entropy=True, top=5)
    grad = o.token_logprobs_bwd(lg, lp.stats, t, lp.logprob)
g.replay()
torch.cuda.synchronize()
rng = torch.tensor([1, 0], device='cuda')
again = o.layer_norm(o.dropout(x, 0.1, rng, residual=x), w, w, residual=x, p=0.1, rng=rng)
assert torch.equal(again.y, out.y) and state.tolist() == [1, 1]
assert torch.equal(o.token_logprobs(lg, t, entropy=True, top=5).entropy, lp.entropy)
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert done.returncode == 0, done.stderr[-2000:]


def test_tensors_of_two_devices_are_refused(ops):
    x = torch.zeros(2, 8, device="cuda")
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.layer_norm(x, torch.ones(8), None)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.token_logprobs(x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.dropout(x, 0.1, _rng())
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.layer_norm(x, None, None, p=0.1, rng=_rng())


def test_the_tuning_setting_leaves_the_row_operators_alone(ops):
    """A process that tunes the compression kernels before its first call of a row operator, and one that does not: the sums of
    the parameter gradients are taken in the same order, which is that of the CTAs that the device holds."""
    import subprocess
    import sys
    code = """
import sys
import torch
from hyc_lora_b200 import _lib, rowops as o
tuned = sys.argv[1] == 'tuned'
digests = []
for dtype, cols in ((torch.bfloat16, 768), (torch.float32, 1024), (torch.bfloat16, 4096)):
    g = torch.Generator().manual_seed(cols)
    dy, z = (torch.randn(5000, cols, generator=g).to(dtype).cuda() for _ in range(2))
    mean, rstd = torch.zeros(5000, device='cuda'), torch.ones(5000, device='cuda')
    for ctas in ((2, 0) if tuned else (0, 0)):
        assert _lib.lib.hyc_set_tuning(0, 0, ctas) == 0
        for t in o.layer_norm_bwd(dy, z, None, mean, rstd, param_dtype=torch.float32)[2:]:
            digests.append(t.view(torch.int32).long().mul(torch.arange(1, cols + 1, device='cuda')).sum().item())
print(digests)
"""
    def digests(how):
        done = subprocess.run([sys.executable, "-c", code, how], capture_output=True, text=True, timeout=300, cwd=ROOT)
        assert done.returncode == 0, done.stderr[-2000:]
        return done.stdout

    assert digests("tuned") == digests("plain")


@pytest.mark.parametrize("which", ["clusters", "norm backward"])
def test_a_refused_launch_is_reported_once(which):
    """Launches into a stream whose capture has been invalidated (on the host, by a synchronisation inside it) are refused by the
    runtime.  That call says so; the next one, on a stream in order, is not blamed for it.  In a process of its own: torch's
    generator does not come out of an invalidated capture."""
    import subprocess
    import sys
    code = """
import ctypes as C
import sys
import torch
from hyc_lora_b200 import _lib
logits, stats = torch.ones(2, 40000, device='cuda'), torch.empty(2, 2, device='cuda')
x, y, one, sums = (torch.ones(n, device='cuda') for n in (384, 384, 64, 768))
rng = torch.tensor([1, 2], device='cuda')

def dropout(stream):
    a = _lib.HycDropoutArgs(rows=1, cols=384, dtype=_lib.HYC_F32, x=x.data_ptr(), y=y.data_ptr(), rng=rng.data_ptr(), p=0.5)
    return _lib.lib.hyc_dropout(C.byref(a), stream)

def norm_backward(stream):
    a = _lib.HycLayerNormBwdArgs(rows=6, cols=64, dtype=_lib.HYC_F32, param_dtype=_lib.HYC_F32, dy=x.data_ptr(), dy_stride=64,
                                 z=x.data_ptr(), z_stride=64, mean=one.data_ptr(), rstd=one.data_ptr(), dresidual=y.data_ptr(),
                                 dbias=one.data_ptr(), partials=sums.data_ptr())
    return _lib.lib.hyc_layer_norm_bwd(C.byref(a), stream)

def clusters(stream):
    a = _lib.HycLogprobArgs(logits=logits.data_ptr(), rows=2, row_stride=40000, seq=2, vocab=40000, dtype=_lib.HYC_F32, stats=stats.data_ptr())
    return _lib.lib.hyc_token_logprobs(C.byref(a), stream)

first = clusters if sys.argv[1] == 'clusters' else norm_backward
good, broken, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
torch.cuda.synchronize()
codes = [first(good.cuda_stream), dropout(good.cuda_stream)]
good.synchronize()
with torch.cuda.stream(broken):
    graph.capture_begin(capture_error_mode='thread_local')
    try:
        broken.synchronize()
        raise SystemExit('a capture outlived a synchronisation')
    except RuntimeError:
        pass
    codes.append(first(broken.cuda_stream))
    try:
        graph.capture_end()
    except RuntimeError:
        pass
codes += [dropout(good.cuda_stream), first(good.cuda_stream)]
good.synchronize()
print(codes)
"""
    done = subprocess.run([sys.executable, "-c", code, which], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert done.returncode == 0 and done.stdout.split("\n")[0] == "[0, 0, -8, 0, 0]", (done.stdout, done.stderr[-2000:])
