"""The host side of drawing, the policy loss and clipping: struct layouts, what
is refused before a device is touched, and the host form of the learn step's
clip."""
import ctypes as C
import math
import subprocess
from dataclasses import replace
from pathlib import Path

import numpy as np
import pytest

from krystal_b200 import abi, policy
from krystal_b200.learn import LearnOptions, UpdatePlan, apply_update
from krystal_b200.model import BRAIN_FORWARD_CONFIG, create_brain_forward_weights
from tests import policy_cases as ref

HEADER = Path(__file__).resolve().parent.parent / "include" / "krystal_cuda.h"
STRUCTS = {"kc_rows_view": "KcRowsView", "kc_sampling": "KcSampling", "kc_draw_out": "KcDrawOut",
           "kc_policy_loss_view": "KcPolicyLossView", "kc_grad_view": "KcGradView"}


def test_struct_layouts_match_the_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for cname, pyname in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        for f, _ in getattr(abi, pyname)._fields_:
            lines.append(f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f.rstrip("_")}));')
    lines.append('printf("max row %u\\n", KC_MAX_ROW); return 0; }')
    (tmp_path / "probe.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "probe"), str(tmp_path / "probe.c")], check=True)
    out = subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout
    want = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}
    for cname, pyname in STRUCTS.items():
        cls = getattr(abi, pyname)
        assert C.sizeof(cls) == want[(cname, "size")], cname
        for f, _ in cls._fields_:
            assert getattr(cls, f).offset == want[(cname, f)], (cname, f)
    assert want[("max", "row")] == abi.KC_MAX_ROW


def test_a_null_handle_is_refused():
    lib = abi.load()
    rows, s = policy.dense_rows(0, "f32", 1, 1), policy.Sampling().device_struct()
    out, loss, grads = abi.KcDrawOut(), abi.KcPolicyLossView(), (abi.KcGradView * 1)()
    calls = [lib.kc_draw_device(None, C.byref(rows), C.byref(s), None, C.byref(out)),
             lib.kc_draw(None, 1, 1, None, C.byref(s), None, C.byref(out)),
             lib.kc_draw_batch(None, C.byref(s), None, C.byref(out)),
             lib.kc_policy_loss(None, C.byref(rows), C.byref(s), C.byref(loss)),
             lib.kc_set_policy(None, None),
             lib.kc_clip_grads(None, C.addressof(grads), 1, 1.0, None, 0, None)]
    assert calls == [abi.KC_ERR_INVALID_ARG] * len(calls)
    assert b"handle is null" in lib.kc_last_error(None)


def test_workspace_grows_with_the_launches():
    lib = abi.load()
    sizes = [lib.kc_clip_workspace(n) for n in (0, 1, 768, 769, 1536, 1537)]
    assert sizes[0] == sizes[1] == sizes[2] and sizes[3] == sizes[4] == 2 * sizes[0] and sizes[5] == 3 * sizes[0]


def test_names_and_lengths_are_checked():
    with pytest.raises(ValueError, match="f8"):
        policy.dense_rows(0, "f8", 1, 1)
    with pytest.raises(ValueError, match="logits"):
        policy.ragged_rows(0, "f32", 1, 1, None, 0, kind="logits")
    s, keep = policy.Sampling(0.5, row_top_k=[1, 2, 3], row_min_p=np.zeros(3)).host_struct(3)
    assert len(keep) == 2 and s.row_top_k and s.row_min_p and not s.row_top_p
    assert keep[0].dtype == np.uint32 and keep[1].dtype == np.float32
    with pytest.raises(ValueError, match="row_top_p"):
        policy.Sampling(row_top_p=[0.5]).host_struct(2)


def test_the_plain_forms_agree_with_a_sort():
    """The reference the GPU tests go by, against a sort written another way."""
    rng = np.random.default_rng(1)
    for trial in range(40):
        n = int(rng.integers(1, 60))
        v = np.round(rng.normal(0, 2, n), 1)  # ties
        k, p = int(rng.integers(0, n + 2)), float(rng.uniform(0.05, 1.1))
        j, pi, logpi = ref.policy(v, 0.7, k, p)
        ranked = sorted(range(n), key=lambda i: (-v[i], i))
        if k:
            ranked = ranked[:k]
        w = {i: math.exp((v[i] - v.max()) / 0.7) for i in ranked}
        total, mass, kept = math.fsum(w.values()), 0.0, []
        for i in ranked:
            if p < 1 and kept and mass >= p * total:
                break
            kept.append(i)
            mass += w[i]
        assert sorted(kept) == j.tolist()
        assert pi.sum() == pytest.approx(1, abs=1e-12) and np.allclose(np.log(pi), logpi, atol=1e-12)
        # dlogp/dv by differences: the gradient of -log pi(a) with advantage 1
        a = int(j[0])
        g = ref.loss((j, pi, logpi), n, a, 1.0, 0.3, 0.7)[3]
        for i in j.tolist():
            f = []
            for d in (1e-5, -1e-5):
                x = (v + d * (np.arange(n) == i))[j] / 0.7
                lp = x - np.log(np.exp(x).sum())
                f.append(-lp[0] + 0.3 * (np.exp(lp) * lp).sum())
            assert abs((f[0] - f[1]) / 2e-5 - g[i]) < 1e-8


@pytest.mark.parametrize("unfreeze_pool", [False, True])
def test_host_update_is_clipped_to_the_actors_norm(unfreeze_pool):
    cfg = BRAIN_FORWARD_CONFIG.with_token_rows(np.arange(64, dtype=np.uint32))
    h = cfg.hidden_size
    rng = np.random.default_rng(3)
    sums = rng.normal(0, 0.01, 2 * h * h + 5 * h)
    plan = UpdatePlan(np.zeros(1), np.ones(1), 4, True, 1, 1, 0.0, 0.0, 0.0, 0.0)
    actor = sums[:2 * h * h + (2 * h if unfreeze_pool else 0)]
    norm = float(np.sqrt((actor ** 2).sum()))
    for limit in (norm * 2, norm / 4, math.inf):
        w, free = (create_brain_forward_weights(cfg, 7) for _ in range(2))
        opts = LearnOptions(unfreeze_pool=unfreeze_pool, max_update_norm=limit)
        assert apply_update(w, sums, plan, opts)[1] is None
        scaled = sums.copy()
        scaled[:actor.size] *= min(1.0, limit / norm)
        assert apply_update(free, scaled, plan, replace(opts, max_update_norm=math.inf))[1] is None
        for a, b in ((w.selector.wq, free.selector.wq), (w.selector.wk, free.selector.wk), (w.pool, free.pool)):
            assert np.abs(a - b).max() <= 2.0 ** -24  # weights below 1: one f32 rounding
        assert np.array_equal(w.value_head_wv, free.value_head_wv)


def test_learn_options_are_checked():
    for bad in (math.nan, -1.0, -math.inf):
        with pytest.raises(ValueError, match="max_update_norm"):
            LearnOptions(max_update_norm=bad)
    with pytest.raises(ValueError, match="max_update_norm"):
        replace(LearnOptions(), max_update_norm=-2.0)
    assert LearnOptions().max_update_norm == math.inf and LearnOptions().sampling is None
