"""The policy loss where factors are not finite or leave f32: rows that must
have no gradient, masked entries, and gradients whose factors overflow."""
import numpy as np
import pytest

from krystal_b200 import policy
from krystal_b200.backend import CudaBrainBackend
from krystal_b200.model import BRAIN_FORWARD_CONFIG, create_brain_forward_weights

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# a row a warp, a row in a CTA's shared memory, a row over a cluster (f32)
LENGTHS = [40, 300, 900, 5000, 20001]
CUTS = [dict(), dict(top_k=7), dict(top_p=0.9)]


@pytest.fixture(scope="module")
def be():
    cfg = BRAIN_FORWARD_CONFIG.with_token_rows(np.arange(64, dtype=np.uint32))
    b = CudaBrainBackend(cfg, create_brain_forward_weights(cfg, 1337), 0)
    yield b
    b.destroy()


def on_gpu(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, dtype))).cuda()


def policy_loss(be, v, dtype, act, adv, weight, temps=None, beta=0.1, cut=None):
    """(loss, logp, entropy, grad in its type) of the rows of v."""
    rows, n = v.shape
    dv, da, dadv, dw = v.cuda(), on_gpu(act, np.int32), on_gpu(adv, np.float32), on_gpu(weight, np.float32)
    dt = on_gpu(temps, np.float32) if temps is not None else None
    lo, lp, h = (torch.full((rows,), 9.0, device="cuda") for _ in range(3))
    grad = torch.full_like(dv, 9.0)
    s = policy.Sampling(**(cut or {}), row_temperature=dt.data_ptr() if dt is not None else None)
    torch.cuda.synchronize()
    be.policy_loss(policy.dense_rows(dv.data_ptr(), dtype, rows, n), s, da.data_ptr(), dadv.data_ptr(), beta,
                   dw.data_ptr(), loss=lo.data_ptr(), logp=lp.data_ptr(), entropy=h.data_ptr(), grad=grad.data_ptr())
    be.synchronize()
    return lo.cpu().numpy(), lp.cpu().numpy(), h.cpu().numpy(), grad.cpu()


@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", LENGTHS)
def test_a_row_without_an_answer_has_no_gradient_whatever_its_factors(be, n, dtype, cut):
    """No target, a target outside the row, a masked one and a temperature of 0,
    each with advantages and weights that are not finite, between rows that
    learn."""
    rng = np.random.default_rng(n)
    nan, inf = np.nan, np.inf
    factors = [(nan, 1.0), (inf, 1.0), (-inf, 2.0), (1.0, nan), (0.5, inf), (nan, nan)]
    kinds = [-1, n + 3, 0, 1]  # of the row's action; entry 0 is masked, entry 1 the largest, at temperature 0
    rows = [(k, a, w) for k in kinds for a, w in factors]
    v = torch.from_numpy(rng.normal(0, 1.5, (len(rows) + 2, n)).astype(np.float32))
    v[:, 1] = v.amax(1) + 0.5
    v[:, 0] = -inf
    act = [1] + [r[0] for r in rows] + [1]
    adv, weight = [0.7] + [r[1] for r in rows] + [-0.4], [1.0] + [r[2] for r in rows] + [1.5]
    temps = [0.8] + [0.0 if r[0] == 1 else 0.8 for r in rows] + [0.8]
    lo, lp, h, g = policy_loss(be, v.to(TYPES[dtype]), dtype, act, adv, weight, temps, cut=cut)
    quiet = slice(1, len(rows) + 1)
    assert (lo[quiet] == 0).all()
    assert bool((g[quiet] == 0).all())
    assert [x for x in lp[quiet]] == [0.0 if r[0] == -1 or r[0] == 1 else -inf for r in rows]
    assert np.isfinite(h).all()
    for i in (0, len(rows) + 1):  # the rows beside them learn
        assert np.isfinite(lo[i]) and lo[i] != 0 and bool(torch.isfinite(g[i]).all()) and float(g[i, 1]) != 0
