"""The global gradient norm and clipping against a plain 64-bit form.

The norm's sums are 64-bit: n squares, each exact to 2^-53, added in some
order, are within n * 2^-53 of their sum (n < 2^24 here: 2^-29), the norm
within half of that. A clipped element is g * scale with the scale rounded to
f32 (2^-24) and the product rounded to f32 and then its type: 2^-24 + 2^-24 +
half a step of the type; f64 elements are one product by an f64 scale.
"""
import math

import numpy as np
import pytest

from krystal_b200 import abi
from krystal_b200.backend import CudaBrainBackend
from krystal_b200.model import BRAIN_FORWARD_CONFIG, create_brain_forward_weights
from krystal_b200.policy import GradList

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}
NORM_TOL = 2.0 ** -29
ELEMENT_TOL = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -11 + 2.0 ** -23, torch.bfloat16: 2.0 ** -8 + 2.0 ** -23,
               torch.float64: 2.0 ** -29}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133, torch.float64: 0.0}


@pytest.fixture(scope="module")
def be():
    cfg = BRAIN_FORWARD_CONFIG.with_token_rows(np.arange(64, dtype=np.uint32))
    b = CudaBrainBackend(cfg, create_brain_forward_weights(cfg, 1337), 0)
    yield b
    b.destroy()


def make(sizes, dtypes, seed=0, offset=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        buf = torch.empty(n + offset, dtype=TYPES[dtypes[i % len(dtypes)]], device="cuda")
        buf.copy_(torch.randn(n + offset, device="cuda", generator=g) * scale * (1 + i % 3))
        out.append(buf[offset:])
    return out


def run(be, grads, max_norm, outs=None, weights=None):
    res = torch.full((2,), -1.0, dtype=torch.float64, device="cuda")
    lst = GradList(grads, outs, weights)
    torch.cuda.synchronize()
    be.clip_grads(lst, max_norm, res.data_ptr())
    be.synchronize()
    return res.tolist()


def want_norm(grads, weights=None):
    weights = weights or [1.0] * len(grads)
    return math.sqrt(math.fsum(w * w * math.fsum((t.double().cpu().numpy() ** 2).tolist())
                               for t, w in zip(grads, weights)))


def check(be, grads, max_norm, outs=None, weights=None):
    before = [t.clone() for t in grads]
    norm = want_norm(grads, weights)
    got = run(be, grads, max_norm, outs, weights)
    assert got[0] == pytest.approx(norm, rel=NORM_TOL)
    scale = max_norm / got[0] if got[0] > max_norm else 1.0
    assert got[1] == pytest.approx(scale, rel=2.0 ** -52)
    for b, o in zip(before, outs if outs is not None else grads):
        want = b.double() * scale
        assert bool(((o.double() - want).abs() <= ELEMENT_TOL[b.dtype] * want.abs() + TINY[b.dtype]).all())
    return got


@pytest.mark.parametrize("dtypes", [["f32"], ["f16"], ["bf16"], ["f64"], ["f32", "bf16", "f64", "f16"]])
@pytest.mark.parametrize("sizes", [[1], [3, 1, 2], [7, 0, 5000], [8191, 8192, 8193, 16384, 16385],
                                   [1 << 20, 5, 300001], [33] * 70])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_clip(be, dtypes, sizes, offset):
    for max_norm in (0.5, 1e9, 0.0):
        grads = make(sizes, dtypes, seed=len(sizes), offset=offset)
        check(be, grads, max_norm)  # in place
        outs = make(sizes, dtypes, seed=9, offset=2 - offset if offset < 3 else 5)
        grads = make(sizes, dtypes, seed=len(sizes), offset=offset)
        keep = [t.clone() for t in grads]
        check(be, grads, max_norm, outs)  # into outputs at another alignment
        assert all(bool((a == b).all()) for a, b in zip(grads, keep))


def test_weights_and_more_tensors_than_one_launch_holds(be):
    sizes = [1 + (i * 37) % 400 for i in range(1700)]
    grads = make(sizes, ["f32", "bf16"], seed=4)
    weights = [0.1 * (i % 7) for i in range(1700)]
    check(be, grads, 3.0, weights=weights)


def test_the_neighbours_of_a_tensor_stay(be):
    buf = torch.full((4000,), 3.0, device="cuda")
    parts = [buf[5:106], buf[111:112], buf[1001:3001]]
    check(be, parts, 1.0)
    rest = torch.ones(4000, dtype=torch.bool, device="cuda")
    for a, b in ((5, 106), (111, 112), (1001, 3001)):
        rest[a:b] = False
    assert bool((buf[rest] == 3.0).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_norm_that_is_not_finite_scales_nothing(be, bad):
    grads = make([1000, 50], ["f32", "f16"])
    grads[1][7] = bad
    keep = [t.clone() for t in grads]
    norm, scale = run(be, grads, 0.1)
    assert not math.isfinite(norm) and scale == 1.0
    assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(grads, keep))


def test_extremes(be):
    # squares outside f32's range, and outside f16's
    big = [torch.full((100,), 3e30, device="cuda"), torch.full((9,), 65504.0, dtype=torch.float16, device="cuda")]
    check(be, big, 1.0)
    small = [torch.full((100,), 1e-30, device="cuda"), torch.full((64,), 2.0 ** -24, dtype=torch.float16, device="cuda")]
    check(be, small, 1e-40)
    zero = [torch.zeros(10, device="cuda")]
    assert run(be, zero, 0.0) == [0.0, 1.0] and not zero[0].any()
    assert run(be, make([5000], ["f32"]), math.inf)[1] == 1.0


def test_a_scale_below_the_smallest_f32(be):
    """One rounding of a 64-bit product is left, which the check's bounds hold."""
    grads = make([5000, 70, 3], ["f32", "bf16", "f64"], scale=1e25)
    outs = [torch.zeros_like(t) for t in grads]
    check(be, grads, 1e-20, outs)
    assert all(bool((o != 0).any()) for o in outs)
    check(be, grads, 1e-20)


def test_equal_calls_give_equal_bits(be):
    grads = make([100003, 77, 65536], ["f32", "bf16"], seed=8)
    outs = [[torch.empty_like(t) for t in grads] for _ in range(3)]
    res = [run(be, grads, 0.7, o) for o in outs]
    assert res[0] == res[1] == res[2]
    assert all(torch.equal(a, b) for o in outs[1:] for a, b in zip(outs[0], o))


def test_captured_clips_replay_side_by_side(be):
    """Two graphs with a list each, replayed at once on two streams."""
    prev, work = be.stream_ptr(), []
    for i in range(2):
        grads = make([50000, 333], ["f32", "f16"], seed=i)
        outs = [torch.empty_like(t) for t in grads]
        res = torch.zeros(2, dtype=torch.float64, device="cuda")
        lst, side, g = GradList(grads, outs), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        be.set_stream(side.cuda_stream)
        try:
            with torch.cuda.graph(g, stream=side):
                be.clip_grads(lst, 2.0, res.data_ptr())
        finally:
            be.set_stream(prev)
        work.append((grads, outs, res, side, g, lst))
    for rep in range(5):
        for grads, *_ in work:
            for t in grads:
                t.mul_(1.5)
        torch.cuda.synchronize()
        for _, _, _, side, g, _ in work:
            with torch.cuda.stream(side):
                g.replay()
        torch.cuda.synchronize()
        for grads, outs, res, *_ in work:
            assert float(res[0]) == pytest.approx(want_norm(grads), rel=NORM_TOL)
            for t, o in zip(grads, outs):
                want = t.double() * float(res[1])
                assert bool(((o.double() - want).abs() <= ELEMENT_TOL[t.dtype] * want.abs() + TINY[t.dtype]).all())
    for w in work:
        w[4].reset()


def test_refusals(be):
    t = torch.ones(8, device="cuda")
    res = torch.zeros(2, dtype=torch.float64, device="cuda")
    lst = GradList([t])
    for bad in (math.nan, -1.0):
        with pytest.raises(abi.KrystalCudaError, match="max_norm"):
            be.clip_grads(lst, bad, res.data_ptr())
    with pytest.raises(abi.KrystalCudaError, match="8-byte"):
        be.clip_grads(lst, 1.0, res.data_ptr() + 4)
    with pytest.raises(abi.KrystalCudaError, match="incomplete"):
        be.clip_grads(lst, 1.0, 0)
    lst.workspace_bytes -= 8
    with pytest.raises(abi.KrystalCudaError, match="workspace"):
        be.clip_grads(lst, 1.0, res.data_ptr())
    lst.workspace_bytes += 8
    for field, value, match in (("dtype", 7, "f32, f16"), ("in_", 0, "null"), ("in_", t.data_ptr() + 2, "aligned"),
                                ("weight", math.inf, "weight"), ("n", 1 << 41, "2\\^40")):
        lst = GradList([t])
        setattr(lst.views[0], field, value)
        with pytest.raises(abi.KrystalCudaError, match=match):
            be.clip_grads(lst, 1.0, res.data_ptr())
    assert bool((t == 1).all())
    with pytest.raises(ValueError, match="contiguous"):
        GradList([torch.ones(4, 4, device="cuda").t()])
    with pytest.raises(ValueError, match="CUDA device"):
        GradList([torch.ones(4)])
    with pytest.raises(ValueError, match="type and size"):
        GradList([t], [t[:4]])
    with pytest.raises(ValueError, match="at least one"):
        GradList([])
    with pytest.raises(ValueError, match="f32, f16"):
        GradList([torch.ones(4, device="cuda", dtype=torch.int32)])
