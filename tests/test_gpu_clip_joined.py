"""The partial sums of a clip where its two launches overlap, and where a list
takes many launches."""
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
