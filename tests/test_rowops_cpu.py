"""No-GPU checks of the row operators: the generator against its published vectors, refusals at the C entry points and in
Python, and the plain 64-bit forms the GPU tests compare with against torch's own."""
import ctypes as C
import glob
import os
import re

import numpy as np
import pytest
import torch

from oracle import rowops_oracle as ro

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hyc_lora_b200", "csrc")


@pytest.fixture(scope="module")
def lib():
    from hyc_lora_b200 import build
    build.build()
    from hyc_lora_b200 import _lib
    return _lib


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_generator_matches_the_published_vectors(counter, key, want):
    got = ro.philox4x32_10(np.array([counter], dtype=np.uint64), key)
    assert tuple(int(v) for v in got[0]) == want


def test_words_of_a_range_are_those_of_the_whole():
    whole = ro.words(2 ** 63 + 5, -3, 64)
    assert np.array_equal(whole[13:40], ro.words(2 ** 63 + 5, -3, 27, first=13))


def test_plain_forms_against_autograd():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 33, dtype=torch.float64, generator=g, requires_grad=True)
    w = torch.randn(33, dtype=torch.float64, generator=g, requires_grad=True)
    b = torch.randn(33, dtype=torch.float64, generator=g, requires_grad=True)
    dy = torch.randn(5, 33, dtype=torch.float64, generator=g)
    y = torch.nn.functional.layer_norm(x, (33,), w, b, 1e-5)
    y.backward(dy)
    (y2, _, mean, rstd), _ = ro.layer_norm(x.detach(), w.detach(), b.detach(), 1e-5)
    (dx, _, dw, db), _ = ro.layer_norm_bwd(dy, x.detach(), w.detach(), mean, rstd)
    for got, want in ((y2, y), (dx, x.grad), (dw, w.grad), (db, b.grad)):
        assert torch.allclose(got, want, rtol=1e-10, atol=1e-12)
    logits = (4 * torch.randn(6, 40, dtype=torch.float64, generator=g)).requires_grad_(True)
    t = torch.randint(0, 40, (6,), generator=g)
    t[2] = -100
    logp = torch.log_softmax(logits, 1)
    h = -(logp.exp() * logp).sum(1)
    best = logp.topk(3, 1)
    got, _ = ro.token_logprobs(logits.detach(), t, top=3)
    want = torch.where(t == -100, 0.0, logp.gather(1, t.clamp_min(0)[:, None])[:, 0])
    assert torch.allclose(got["logprob"], want) and torch.allclose(got["entropy"], h)
    assert torch.equal(got["top_index"], best.indices) and torch.allclose(got["top_logprob"], best.values)
    d1, d2, d3 = (torch.randn(s, dtype=torch.float64, generator=g) for s in ((6,), (6,), (6, 3)))
    ((want * d1).sum() + (h * d2).sum() + (best.values * d3).sum()).backward()
    grad, _ = ro.token_logprobs_bwd(logits.detach(), got["stats"], t, d1, entropy=got["entropy"], d_entropy=d2,
                                    top_index=got["top_index"], d_top=d3)
    assert torch.allclose(grad, logits.grad, rtol=1e-9, atol=1e-12)


# ------------------------------------------------------------------------------------------------ refusals at the C entries

def _dropout(lib, **kw):
    a = lib.HycDropoutArgs()
    a.rows, a.cols, a.dtype, a.p = 4, 100, lib.HYC_BF16, 0.1
    a.x, a.y, a.rng, a.x_stride = 0x1000, 0x2000, 0x3000, 100
    for k, v in kw.items():
        setattr(a, k, v)
    return lib.lib.hyc_dropout(C.byref(a), None)


def test_dropout_refusals(lib):
    assert lib.lib.hyc_dropout(None, None) == -1
    assert lib.lib.hyc_strerror(-10) == b"a scalar argument is out of its range"
    for bad, code in (({"x": None}, -1), ({"y": None}, -1), ({"rng": None}, -1), ({"rows": -1}, -2), ({"cols": -1}, -2),
                      ({"rows": 2 ** 40, "cols": 2 ** 30}, -2), ({"x_stride": -1}, -2), ({"residual_stride": -1}, -2),
                      ({"dtype": 2}, -4), ({"x": 0x1001}, -6), ({"y": 0x2001}, -6), ({"residual": 0x1001}, -6), ({"rng": 0x3004}, -6),
                      ({"dtype": 0, "x": 0x1002}, -6), ({"p": -0.1}, -10), ({"p": 1.1}, -10), ({"p": float("nan")}, -10)):
        assert _dropout(lib, **bad) == code, bad
    assert _dropout(lib, rows=0, x=None, y=None, rng=None) == 0
    assert _dropout(lib, cols=0) == 0
    assert lib.lib.hyc_rng_take(None, 0x1000, None) == -1 and lib.lib.hyc_rng_take(0x1000, None, None) == -1
    assert lib.lib.hyc_rng_take(0x1004, 0x1000, None) == -6


def _norm(lib, **kw):
    a = lib.HycLayerNormArgs()
    a.rows, a.cols, a.dtype, a.param_dtype, a.eps = 4, 100, lib.HYC_BF16, lib.HYC_F32, 1e-5
    a.x, a.x_stride, a.y, a.mean, a.rstd = 0x1000, 100, 0x2000, 0x3000, 0x3100
    for k, v in kw.items():
        setattr(a, k, v)
    return lib.lib.hyc_layer_norm(C.byref(a), None)


def _norm_bwd(lib, **kw):
    a = lib.HycLayerNormBwdArgs()
    a.rows, a.cols, a.dtype, a.param_dtype = 4, 100, lib.HYC_BF16, lib.HYC_F32
    a.dy, a.dy_stride, a.z, a.z_stride, a.mean, a.rstd, a.dresidual = 0x1000, 100, 0x2000, 100, 0x3000, 0x3100, 0x4000
    for k, v in kw.items():
        setattr(a, k, v)
    return lib.lib.hyc_layer_norm_bwd(C.byref(a), None)


def test_layer_norm_refusals(lib):
    assert lib.lib.hyc_layer_norm(None, None) == -1 and lib.lib.hyc_layer_norm_bwd(None, None) == -1
    for bad, code in (({"x": None}, -1), ({"y": None}, -1), ({"mean": None}, -1), ({"rstd": None}, -1), ({"p": 0.5}, -1),
                      ({"rows": -1}, -2), ({"cols": 0}, -2), ({"cols": -5}, -2), ({"x_stride": -1}, -2), ({"cols": 16385}, -7), ({"rows": 2 ** 31}, -7),
                      ({"dtype": 3}, -4), ({"param_dtype": 3}, -4), ({"x": 0x1001}, -6), ({"z": 0x1001}, -6), ({"weight": 0x1002}, -6),
                      ({"bias": 0x1002}, -6), ({"mean": 0x3002}, -6), ({"p": 0.5, "rng": 0x1004}, -6), ({"p": -1.0}, -10),
                      ({"p": float("nan")}, -10)):
        assert _norm(lib, **bad) == code, bad
    for bad, code in (({"dy": None}, -1), ({"z": None}, -1), ({"mean": None}, -1), ({"dresidual": None}, -1),
                      ({"p": 0.5, "rng": 0x1000}, -1), ({"p": 0.5, "dx": 0x1000}, -1), ({"dweight": 0x1000}, -1), ({"dbias": 0x1000}, -1),
                      ({"dy_stride": -1}, -2), ({"cols": 0}, -2), ({"cols": 16385}, -7), ({"rows": 2 ** 31}, -7), ({"dtype": 3}, -4), ({"dz": 0x1001}, -6),
                      ({"dweight": 0x1002, "partials": 0x1000}, -6), ({"dweight": 0x1000, "partials": 0x1008}, -6), ({"p": 2.0}, -10)):
        assert _norm_bwd(lib, **bad) == code, bad
    assert _norm(lib, rows=0, x=None, y=None, mean=None, rstd=None) == 0
    assert _norm_bwd(lib, rows=0, dy=None, z=None) == 0
    assert lib.lib.hyc_layer_norm_bwd_scratch_floats(-1, 100) == -2
    assert lib.lib.hyc_layer_norm_bwd_scratch_floats(5, 0) == -2
    assert lib.lib.hyc_layer_norm_bwd_scratch_floats(5, 16385) == -7
    assert lib.lib.hyc_layer_norm_bwd_scratch_floats(5, 100) >= 200


def _logprob(lib, **kw):
    a = lib.HycLogprobArgs()
    a.logits, a.rows, a.row_stride, a.seq, a.vocab, a.dtype, a.ignore_index = 0x1000, 4, 100, 4, 100, lib.HYC_BF16, -100
    a.targets, a.logprob, a.stats = 0x2000, 0x3000, 0x4000
    for k, v in kw.items():
        setattr(a, k, v)
    return lib.lib.hyc_token_logprobs(C.byref(a), None)


def _logprob_bwd(lib, **kw):
    a = lib.HycLogprobBwdArgs()
    a.logits, a.rows, a.row_stride, a.seq, a.vocab, a.dtype, a.ignore_index = 0x1000, 4, 100, 4, 100, lib.HYC_BF16, -100
    a.targets, a.d_logprob, a.stats, a.grad = 0x2000, 0x3000, 0x4000, 0x5000
    for k, v in kw.items():
        setattr(a, k, v)
    return lib.lib.hyc_token_logprobs_bwd(C.byref(a), None)


def test_logprob_refusals(lib):
    assert lib.lib.hyc_token_logprobs(None, None) == -1 and lib.lib.hyc_token_logprobs_bwd(None, None) == -1
    common = (({"logits": None}, -1), ({"stats": None}, -1), ({"rows": -1}, -2), ({"vocab": 0}, -2), ({"seq": 0}, -2),
              ({"row_stride": -1}, -2), ({"batch_stride": -1}, -2), ({"top": -1}, -2), ({"vocab": 262145}, -7), ({"rows": 2 ** 31}, -7), ({"dtype": 2}, -4),
              ({"logits": 0x1001}, -6), ({"targets": 0x2004}, -6), ({"stats": 0x4004}, -6))
    for bad, code in common + (({"logprob": None}, -1), ({"top": 5}, -1), ({"top": 101}, -2), ({"top": 33}, -7),
                               ({"top": 5, "top_index": 0x1004, "top_logprob": 0x1000}, -6), ({"entropy": 0x1002}, -6)):
        assert _logprob(lib, **bad) == code, bad
    for bad, code in common + (({"grad": None}, -1), ({"targets": None}, -1), ({"d_entropy": 0x1000}, -1), ({"d_top": 0x1000, "top": 2}, -1),
                               ({"grad": 0x5001}, -6)):
        assert _logprob_bwd(lib, **bad) == code, bad
    assert _logprob(lib, rows=0, logits=None, stats=None) == 0
    assert _logprob_bwd(lib, rows=0, logits=None) == 0


# ------------------------------------------------------------------------------------------------ refusals in Python

def test_packed_records_have_the_layout_of_the_ctypes_ones(lib):
    from hyc_lora_b200 import rowops
    codes = {C.c_int64: "q", C.c_int32: "i", C.c_void_p: "P", C.c_float: "f", C.c_double: "d"}
    for packer, record in ((rowops._DROPOUT, lib.HycDropoutArgs), (rowops._LAYER_NORM, lib.HycLayerNormArgs),
                           (rowops._LAYER_NORM_BWD, lib.HycLayerNormBwdArgs), (rowops._LOGPROB, lib.HycLogprobArgs),
                           (rowops._LOGPROB_BWD, lib.HycLogprobBwdArgs)):
        assert packer.format == "@" + "".join(codes[kind] for _, kind in record._fields_)
        assert packer.size == C.sizeof(record)


def test_python_refuses_cpu_tensors_and_wrong_arguments(lib):
    from hyc_lora_b200 import rowops
    x, rng = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: rowops.dropout(x, 0.1, rng), lambda: rowops.layer_norm(x, None, None), lambda: rowops.token_logprobs(x),
                 lambda: rowops.rng_take(rng), lambda: rowops.layer_norm_bwd(x, x, None, x, x),
                 lambda: rowops.token_logprobs_bwd(x, x)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(ValueError, match="rng must be"):
        rowops.dropout(x, 0.1, torch.zeros(2))
    with pytest.raises(ValueError, match="rng must be"):
        rowops.rng_take(torch.zeros(3, dtype=torch.int64))


def test_modules_validate_and_keep_their_state(lib):
    from hyc_lora_b200.operators.efficient_dropout import EfficientMemoryCounterDropout
    from hyc_lora_b200.operators.efficient_layernorm import EfficientMemoryDropoutAddLayerNorm
    from hyc_lora_b200.operators.efficient_logprob import token_cross_entropy
    for p in (-0.1, 1.5):
        with pytest.raises(ValueError):
            EfficientMemoryCounterDropout(p)
        with pytest.raises(ValueError):
            EfficientMemoryDropoutAddLayerNorm(8, p=p)
    with pytest.raises(ValueError):
        EfficientMemoryDropoutAddLayerNorm((4, 8))
    with pytest.raises(ValueError, match="reduction"):
        token_cross_entropy(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64), reduction="avg")
    m = EfficientMemoryCounterDropout(0.1, seed=7)
    assert m.rng_state.tolist() == [7, 0] and "rng_state" in m.state_dict()
    x = torch.ones(3, 4)
    assert m.eval()(x) is x and torch.equal(m(x, x), 2 * x)
    torch.manual_seed(5)
    a = EfficientMemoryCounterDropout(0.1).rng_state.clone()
    torch.manual_seed(5)
    assert torch.equal(a, EfficientMemoryCounterDropout(0.1).rng_state)
    n = EfficientMemoryDropoutAddLayerNorm(8, p=0.1)
    assert isinstance(n, torch.nn.LayerNorm) and "rng_state" in n.state_dict()
    assert "rng_state" not in EfficientMemoryDropoutAddLayerNorm(8).state_dict()
    with pytest.raises(ValueError, match="last dimension"):
        n(torch.zeros(2, 9))


@pytest.mark.parametrize("p,training", [(0.1, False), (0.0, True), (0.0, False)])
def test_counter_dropout_takes_the_same_residuals_without_dropping(lib, p, training):
    """With dropout the kernel refuses a residual of another shape or dtype; so does the sum that takes its place."""
    from hyc_lora_b200.operators.efficient_dropout import EfficientMemoryCounterDropout
    m = EfficientMemoryCounterDropout(p).train(training)
    x = torch.ones(3, 4)
    for bad in (torch.ones(1, 4), torch.ones(4), torch.ones(3, 1), torch.ones(2, 3, 4)):
        with pytest.raises(ValueError, match="residual has shape"):
            m(x, bad)
    for bad in (torch.ones(3, 4, dtype=torch.bfloat16), torch.ones(3, 4, dtype=torch.float64)):
        with pytest.raises(TypeError, match="residual is"):
            m(x, bad)
    assert torch.equal(m(x, 2 * x), 3 * x) and m(x) is x


def test_replacement_leaves_the_row_operators_alone(lib):
    from hyc_lora_b200.hosts.replace import replace_module, uniform_config
    from hyc_lora_b200.operators.efficient_dropout import EfficientMemoryCounterDropout
    from hyc_lora_b200.operators.efficient_layernorm import EfficientMemoryDropoutAddLayerNorm
    model = torch.nn.ModuleDict({"norm": EfficientMemoryDropoutAddLayerNorm(128, p=0.1), "drop": EfficientMemoryCounterDropout(0.1)})
    assert replace_module(model, uniform_config()) == 0
    assert type(model["norm"]) is EfficientMemoryDropoutAddLayerNorm


def test_hosts_build_with_and_without_the_row_operators(lib):
    from hyc_lora_b200.hosts.roberta import EncoderClassifier, EncoderConfig
    from hyc_lora_b200.operators.efficient_layernorm import EfficientMemoryDropoutAddLayerNorm
    small = dict(hidden=32, layers=1, heads=2, ffn=64, vocab=50, max_pos=40, lora_r=4)
    plain = EncoderClassifier(EncoderConfig(**small), device="cpu", init_on_cpu=True)
    assert type(plain.layers[0].out_LayerNorm) is torch.nn.LayerNorm and plain.emb_dropout is None
    joined = EncoderClassifier(EncoderConfig(hidden_dropout=0.1, **small), device="cpu", init_on_cpu=True)
    assert type(joined.layers[0].out_LayerNorm) is EfficientMemoryDropoutAddLayerNorm
    for (a, p), (b, q) in zip(plain.named_parameters(), joined.named_parameters()):
        assert a == b and torch.equal(p, q)          # the same weights from the same seed
    ids, labels = torch.randint(0, 50, (2, 7)), torch.tensor([0, 1])
    assert torch.isfinite(plain(ids, labels))


def test_calibration_kept_puts_every_site_back(lib):
    from hyc_lora_b200.operators import _common as co
    from hyc_lora_b200.operators.efficient_gemm import EfficientMemoryGEMM
    from hyc_lora_b200.operators.efficient_linear import EfficientMemoryLinear
    from hyc_lora_b200.operators.efficient_softmax import EfficientMemorySoftmax
    model = torch.nn.ModuleList([EfficientMemoryLinear(128, 8, rank=0, outlier_mode="channel"), EfficientMemoryGEMM(), EfficientMemorySoftmax(0.05)])
    linear, gemm, softmax = model
    one = [torch.ones(2, 2) for _ in range(4)]
    co.update_static(gemm.static_value_1, 0, *one)
    gemm.static_value_1.cache["pool_density"] = 0.25
    gemm.iteration = 1
    linear.site.calib.score = torch.arange(4.0)
    before = [co.calibration_state_dict(m) for m in model]

    def pass_over_other_data():
        for m in model:
            m.iteration += 2
        for static in (linear.static_value, gemm.static_value_1, gemm.static_value_2):
            co.update_static(static, 0, *(2 * t for t in one))
            static.cache["pool_density"] = 0.5
        softmax.static_value = torch.ones(())
        linear.site.calib.score, linear.site.calib.channels = torch.zeros(4), torch.zeros(1, dtype=torch.int32)
        linear.site.calib._compared = linear.site.calib.channels
        linear.site.output_format, linear.site.pending_output = (4, 0, 0, linear.site.calib), object()
        co._shared.insert(0, "a record")
        co._last_norm_output = "an output"

    shared, last, static = list(co._shared), co._last_norm_output, gemm.static_value_1
    for fails in (False, True):
        try:
            with co.calibration_kept(model):
                pass_over_other_data()
                assert linear.iteration == 2
                if fails:
                    raise KeyError
        except KeyError:
            pass
        after = [co.calibration_state_dict(m) for m in model]
        assert str(before) == str(after)
        assert gemm.static_value_1 is static and static.cache == {"pool_density": 0.25} and linear.static_value.cache == {}
        assert linear.site.output_format is None and linear.site.pending_output is None and not hasattr(linear.site.calib, "_compared")
        assert co._shared == shared and co._last_norm_output is last


# ------------------------------------------------------------------------------------------------ orderings, read from the source

def _kernel_bodies(text):
    """(name, body) of every __global__ function of a source file."""
    for found in re.finditer(r"__global__ void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\(", text):
        at = text.index("{", found.end())
        depth, end = 1, at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        yield found.group(1), text[at:end]


def test_ctas_of_a_cluster_meet_before_they_write_into_one_another():
    """Another CTA's shared memory may be accessed only after it is known to have started: a wait at a cluster barrier stands
    in front of the first store, and one behind the last in front of the exit."""
    seen = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        text = open(path).read()
        for name, body in _kernel_bodies(text):
            stores = [m.start() for m in re.finditer(r"\b(?:ld|st|red|atom)\.(?:\w+\.)*shared::cluster\.", body)]
            if not stores:
                continue
            seen += 1
            waits = [m.start() for m in re.finditer(r"\bcluster_(?:wait|barrier)\(\)", body)]
            assert waits and waits[0] < stores[0] and waits[-1] > stores[-1], (path, name)
            if body[waits[0]:].startswith("cluster_wait"):
                assert 0 <= body.find("cluster_arrive()") < waits[0], (path, name)
    assert seen >= 1
