"""The partial sums of a clip where its two launches overlap, and where a list
takes many launches."""
import math

import numpy as np
import pytest

from krystal_b200.backend import CudaBrainBackend
from krystal_b200.model import BRAIN_FORWARD_CONFIG, create_brain_forward_weights
from krystal_b200.policy import GradList

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def be():
    cfg = BRAIN_FORWARD_CONFIG.with_token_rows(np.arange(64, dtype=np.uint32))
    b = CudaBrainBackend(cfg, create_brain_forward_weights(cfg, 1337), 0)
    yield b
    b.destroy()


@pytest.mark.parametrize("n", [100, 50_000, 9_000_000])
def test_a_clip_sees_its_own_partial_sums(be, n):
    """Two lists that share a workspace, clipped in turn without a wait: a sum
    left by the other one would show in the norm."""
    g = [torch.randn(n, device="cuda") * s for s in (1.0, 3.0)]
    outs = [torch.empty_like(x) for x in g]
    lists = [GradList([x], [o]) for x, o in zip(g, outs)]
    lists[1].workspace = lists[0].workspace
    want = [float(x.double().norm()) for x in g]
    res = torch.zeros(60, 2, dtype=torch.float64, device="cuda")
    torch.cuda.synchronize()
    for i in range(60):
        be.clip_grads(lists[i % 2], 0.5, res[i].data_ptr())
    be.synchronize()
    for k in range(2):
        mine = res[k::2]
        assert torch.equal(mine, mine[:1].expand_as(mine))
        assert abs(float(mine[0, 0]) - want[k]) <= want[k] * 2.0 ** -28  # 2^-29 each side: n below 2^24
        assert abs(float(outs[k].double().norm()) - 0.5) <= 2.0 ** -22  # an element is off by 2^-23


@pytest.mark.parametrize("count", [768, 769, 1536, 1537, 5000])
@pytest.mark.parametrize("share", [0.3, 2.0])
def test_lists_of_many_launches(be, count, share):
    """One norm and one scale over all of a list's launches, in place and into
    other tensors, with empty tensors among them."""
    gen = torch.Generator(device="cuda").manual_seed(count)
    flat = torch.randn(count * 40, device="cuda", generator=gen)
    sizes = [(i * 7) % 41 for i in range(count)]
    grads = [flat[i * 40:i * 40 + min(n, 40)] for i, n in enumerate(sizes)]
    before = [g.clone() for g in grads]
    norm = float(torch.cat(grads).double().norm())
    out = torch.full_like(flat, 7.0)
    outs = [out[i * 40:i * 40 + min(n, 40)] if i % 3 else g for i, (g, n) in enumerate(zip(grads, sizes))]
    res = torch.zeros(2, dtype=torch.float64, device="cuda")
    lst = GradList(grads, outs)
    torch.cuda.synchronize()
    be.clip_grads(lst, norm * share, res.data_ptr())
    be.synchronize()
    got, scale = res.tolist()
    assert abs(got - norm) <= norm * 2.0 ** -30  # both sums of fewer than 2^18 squares in 64 bits
    assert scale == (norm * share / got if share < 1 else 1.0)
    for b, o in zip(before, outs):
        want = b.double() * scale
        assert bool(((o.double() - want).abs() <= 2.0 ** -23 * want.abs()).all())  # two half steps: scale, product


def clip_time(be, count):
    """The least device time of a clip of `count` tensors of 4 elements."""
    flat = torch.ones(count, 4, device="cuda")
    lst, res = GradList(list(flat.unbind(0))), torch.zeros(2, dtype=torch.float64, device="cuda")
    stream = torch.cuda.ExternalStream(be.stream_ptr())
    torch.cuda.synchronize()
    times = []
    for _ in range(6):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record(stream)
        be.clip_grads(lst, math.inf, res.data_ptr())
        b.record(stream)
        b.synchronize()
        times.append(a.elapsed_time(b))
    assert res.tolist() == [math.sqrt(4.0 * count), 1.0]
    return min(times[1:])


def test_the_time_of_a_long_list_grows_with_its_length(be):
    """Eight times as many tensors are eight times as many launches; partial sums
    added up by every CTA of every launch would grow with the square."""
    short, long = clip_time(be, 32768), clip_time(be, 262144)
    print(f"32768 tensors: {short:.3f} ms, 262144: {long:.3f} ms")
    assert long < 12 * short


def test_a_sum_of_squares_beyond_f64_scales_nothing(be):
    """Finite f64 gradients whose squares are not: the norm is infinite, and what
    follows sees the gradients as they are."""
    for size, weight in ((1e200, 1.0), (1e100, 1e100)):
        g = torch.full((1000,), size, dtype=torch.float64, device="cuda")
        out, res = torch.zeros_like(g), torch.zeros(2, dtype=torch.float64, device="cuda")
        lst = GradList([g], [out], [weight])
        torch.cuda.synchronize()
        be.clip_grads(lst, 1.0, res.data_ptr())
        be.synchronize()
        assert res.tolist() == [math.inf, 1.0] and torch.equal(out, g)
