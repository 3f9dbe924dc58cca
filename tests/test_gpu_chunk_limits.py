"""Chunk attention over pages whose V scales lie anywhere in float32's range, and infinite values with weights that vanish beside others',
for the kernel of few query rows and that of many."""
import numpy as np
import pytest

from test_gpu_chunk_attention import Case, _t

pytestmark = pytest.mark.gpu

# B, L, Hq, Hkv, W: few rows a KV head, and so many rows of so many KV heads that these go to the kernel of many
FEW, MANY = (2, 3, 8, 2, 40), (32, 64, 16, 4, 25)
TAG = {"int8": 1, "fp8": 3, "int4": 4, "int4r": 5}


def _case(seed, shape, D, mix, q_dtype="float32", **kw):
    B, L, Hq, Hkv, W = shape
    return Case(seed, B, L, Hq, Hkv, D, W, mix, q_dtype, scale_dtype=np.float32, **kw)


def _upload(s, *names):
    for n in names or tuple(s.host):
        setattr(s.pools, n, _t(s.host[n]))


def _check_some(s, out_dtype=None, some=2, **kw):
    """The first sequences' outputs alone (the oracle is slow)."""
    import torch
    got = s.run(out_dtype=None if out_dtype is None else getattr(torch, out_dtype), **kw)
    keep = {n: getattr(s, n) for n in ("table", "counts", "valid", "q_lens", "q")}
    for n, x in keep.items():
        setattr(s, n, None if x is None else x[:some])
    s.check(got[:some], **{n: x for n, x in kw.items() if n in ("causal", "sm_scale")})
    for n, x in keep.items():
        setattr(s, n, x)
    return got


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", [FEW, MANY])
@pytest.mark.parametrize("mix", ["bytes", "all"])
def test_a_step_of_tiny_pages_between_ordinary_ones(mix, shape, D):
    s = _case(1, shape, D, mix, "float16")
    W = shape[-1]
    s.tags[:] = s.rng.choice([1, 3] if mix == "bytes" else [1, 3, 4, 5], s.NP)
    for first, size in ((8, 1e-37), (16, 1e-25)):
        for n, x in s.host.items():
            if n.startswith("v_") and n.endswith("_scale"):
                x[s.table[:, :, first:first + 8]] = size
    _upload(s)
    assert W >= 24
    for out in ("float32", "bfloat16"):
        _check_some(s, out)
    _check_some(s, "float32", splits=2)


def _largest(s, kind):
    """|V| of no page is larger."""
    code = {"int8": 128, "fp8": 448, "int4": 8, "int4r": 16}[kind]
    return code * float(np.abs(s.host[f"v_{kind}_scale"]).max())


def _far(power, kind, shape, D, **kw):
    """V's scales times 2^power: outputs times 2^power."""
    import torch
    s = _case(abs(power), shape, D, kind)
    s.tags[:] = TAG[kind]
    near = _check_some(s, "float32", **kw)
    size = _largest(s, kind)
    n = f"v_{kind}_scale"
    s.host[n] = np.ldexp(s.host[n], power).astype(np.float32)
    assert (s.host[n] >= 2.0 ** -126).all()
    _upload(s, n)
    got = s.run(out_dtype=torch.float32, **kw).double()
    assert torch.isfinite(got).all()
    # A weight's exponent has the logarithm of the scale: below 2^7, so rounded by 2^-18 and off by 2^-17 of its own, and three
    # roundings of sums of that size: 3 2^-17 in all, times ln 2, in either run; the rest is as small as a weight's two parts.
    error = float((torch.ldexp(got, torch.tensor(-power, device=got.device)) - near.double()).abs().amax())
    assert error <= 2 * 3 * 2.0 ** -17 * size, (error, size)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", [FEW, MANY])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("power", [-110, -70, 70])
def test_scales_far_from_one(power, kind, shape, D):
    _far(power, kind, shape, D)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", [FEW, MANY])
@pytest.mark.parametrize("kind", ["int4", "int4r"])
@pytest.mark.parametrize("power", [-110, -70, 70])
def test_scales_far_from_one_of_4_bits(power, kind, shape, D):
    _far(power, kind, shape, D)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", [FEW, MANY])
@pytest.mark.parametrize("kind", ["int4", "int4r"])
@pytest.mark.parametrize("power", [-70, 70])
def test_key_scales_far_from_one_of_4_bits(power, kind, shape, D):
    import torch
    s = _case(abs(power), shape, D, kind)
    s.tags[:] = TAG[kind]
    near = s.run(out_dtype=torch.float32, sm_scale=0.125)
    n = f"k_{kind}_scale"
    s.host[n] = np.ldexp(s.host[n], power).astype(np.float32)
    _upload(s, n)
    got = s.run(out_dtype=torch.float32, sm_scale=float(np.ldexp(0.125, -power)))
    assert torch.equal(got, near)                                # powers of two cancel


@pytest.mark.parametrize("shape", [FEW, MANY])
def test_infinite_scales_beside_large_ones(shape):
    """Of a page's groups one is infinite, the others past float16's range."""
    s = _case(6, shape, 128, "int4")
    s.tags[:] = TAG["int4"]
    page = s.table[:, :, 2].ravel()
    s.host["v_int4_scale"][page] = 1e5
    s.host["v_int4_scale"][page, 1] = -np.inf
    _upload(s)
    _check_some(s, "float32")
    _check_some(s, "float32", splits=2)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", [FEW, MANY])
@pytest.mark.parametrize("kind", ["int8", "fp8", "int4", "int4r"])
@pytest.mark.parametrize("splits", [1, 3])
def test_values_next_to_the_ranges_end(splits, kind, shape, D):
    """The weighted sums, before they are divided, are past float32's range."""
    _far({"int8": 124, "fp8": 122, "int4": 124, "int4r": 124}[kind], kind, shape, D, splits=splits)


@pytest.mark.parametrize("shape", [FEW, MANY])
def test_scales_at_the_ranges_end(shape):
    """Scales from 2^126 on, whose inverse is below the normal range."""
    import torch
    s = _case(5, shape, 64, "int8")
    s.tags[:] = 1
    s.host["v_int8"] = (s.host["v_int8"] % 3 - 1).astype(np.int8)
    s.host["v_int8_scale"][:] = np.float32(1.5 * 2.0 ** -7)
    _upload(s)
    near = _check_some(s, "float32")
    for size in (1.5 * 2.0 ** 127, 1.5 * 2.0 ** 126):
        s.host["v_int8_scale"][:] = np.float32(size)
        _upload(s, "v_int8_scale")
        got = s.run(out_dtype=torch.float32).double() / size
        assert float((got - near.double() / (1.5 * 2.0 ** -7)).abs().amax()) <= 2 * 3 * 2.0 ** -17


@pytest.mark.parametrize("shape", [FEW, MANY])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("mix", ["fp16", "all"])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_infinite_values_with_weights_that_vanish(value, mix, splits, shape):
    """Scores of some pages are hundreds above those of the page with the infinity, in other waves' and other parts' shares."""
    s = _case(3, shape, 64, mix, ragged=False)
    B, L, Hq, Hkv, W = shape
    s.q[:] = 0
    s.q[..., 0] = 8.0
    s.tags[:] = 0
    s.host["k_fp16"][:] = 0
    for e in range(W):
        s.host["k_fp16"][s.table[:, :, e].ravel(), :, 0] = 400.0 if e >= W // 2 else -400.0
    at = s.table[:, :, 1].ravel()
    s.host["v_fp16"][at, 3, 5] = value
    _upload(s, "k_fp16", "v_fp16")
    _check_some(s, splits=splits)
    _check_some(s, causal=False, splits=splits)
    # and the other way round: what is infinite outweighs the rest
    s.host["k_fp16"][:, :, 0] *= -1
    _upload(s, "k_fp16")
    _check_some(s, splits=splits)


@pytest.mark.parametrize("shape,mix", [(FEW, "all"), (MANY, "all"), (MANY, "fp16")])
def test_runs_repeat_themselves(shape, mix):
    import torch
    s = _case(4, shape, 128, mix, "float16")
    for splits in (0, 3):
        first = s.run(splits=splits)
        for _ in range(3):
            assert torch.equal(first, s.run(splits=splits))
