"""The host side of the bank cache: struct layouts, the storage's size, and what
is refused before a device is touched."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from krystal_b200 import BankCache, abi
from krystal_b200 import cache as kc
from tests import cache_cases as ref

HEADER = Path(__file__).resolve().parent.parent / "include" / "krystal_cuda.h"
STRUCTS = {"kc_cache_view": "KcCacheView", "kc_page_table": "KcPageTable", "kc_cache_rows": "KcCacheRows",
           "kc_question_view": "KcQuestionView", "kc_attend_view": "KcAttendView", "kc_bank_view": "KcBankView",
           "kc_bank_out": "KcBankOut"}


def test_struct_layouts_match_the_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {"]
    for cname, pyname in STRUCTS.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        for f, _ in getattr(abi, pyname)._fields_:
            lines.append(f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));')
    lines.append('printf("page rows %u\\nselect rows %u\\n", KC_CACHE_PAGE, KC_CACHE_MAX_SELECT); return 0; }')
    (tmp_path / "probe.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "probe"), str(tmp_path / "probe.c")], check=True)
    out = subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout
    want = {tuple(line.split()[:2]): int(line.split()[2]) for line in out.splitlines()}
    for cname, pyname in STRUCTS.items():
        cls = getattr(abi, pyname)
        assert C.sizeof(cls) == want[(cname, "size")], cname
        for f, _ in cls._fields_:
            assert getattr(cls, f).offset == want[(cname, f)], (cname, f)
    assert want[("page", "rows")] == abi.KC_CACHE_PAGE == ref.PAGE
    assert want[("select", "rows")] == abi.KC_CACHE_MAX_SELECT


@pytest.mark.parametrize("heads,dim", [(1, 32), (4, 32), (8, 128), (3, 64)])
def test_the_storage_is_two_cells_a_head_and_the_bounds(heads, dim):
    cell = 32 * (2 * dim + 8)
    assert BankCache.bytes_for(7, heads, dim) == 7 * heads * (2 * cell + 2 * dim * 4)
    assert BankCache.bytes_for(1 << 20, 128, 128) > 1 << 40  # past 32 bits


def test_a_null_handle_is_refused():
    lib = abi.load()
    cache, table = abi.KcCacheView(), abi.KcPageTable()
    rows, ask, view = abi.KcCacheRows(), abi.KcQuestionView(), abi.KcAttendView()
    c, t = C.byref(cache), C.byref(table)
    calls = [lib.kc_cache_write(None, c, t, C.byref(rows)), lib.kc_cache_read(None, c, t, None, C.byref(rows)),
             lib.kc_cache_blocks(None, c, t, C.byref(ask), 1, 0, None),
             lib.kc_cache_attend(None, c, t, C.byref(ask), C.byref(view)),
             lib.kc_cache_scores(None, c, t, C.byref(ask), None, None, 0.0, None),
             lib.kc_bank_turn(None, C.byref(abi.KcBatchView()), C.byref(abi.KcBankView()), None,
                              C.byref(abi.KcBankOut()))]
    assert calls == [abi.KC_ERR_INVALID_ARG] * len(calls)
    assert b"handle is null" in lib.kc_last_error(None)
    assert lib.kc_cache_attend_workspace(None, c, t, C.byref(ask), 0) == 0


def test_what_a_cache_cannot_be_is_refused():
    torch = pytest.importorskip("torch")
    with pytest.raises(ValueError, match="cache format"):
        BankCache(1, format="fp4")
    for bad in (dict(pages=0), dict(pages=1, kv_heads=0), dict(pages=1, kv_heads=129), dict(pages=1, head_dim=48)):
        with pytest.raises(ValueError, match="at least one page"):
            BankCache(**bad)
    size = BankCache.bytes_for(2)
    for storage in (torch.zeros(size, dtype=torch.uint8), torch.zeros(size // 4, dtype=torch.float32)):
        with pytest.raises(ValueError, match="CUDA tensor of uint8"):
            BankCache(2, storage=storage)
    with pytest.raises(ValueError, match="element type"):
        kc.cache_rows(0, 0, "i4", 1)
    with pytest.raises(ValueError, match="element type"):
        kc.questions(0, "i4", 1, 1)


def test_the_plain_form_of_the_tests_quantises_as_defined():
    """The reference itself, on values worked out by hand."""
    x = np.array([[127.0, -63.5, 0.5, 1.5, -2.5, 0.0], [0.0] * 6, [np.nan, np.inf, -np.inf, 1.0, 0.0, 0.0]])
    y = ref.quantised(x, "i8")
    assert y[0].tolist() == [127.0, -64.0, 0.0, 2.0, -2.0, 0.0]
    assert (y[1] == 0).all()
    assert y[2, 0] == 0 and y[2, 1] == -y[2, 2] and np.isfinite(y[2]).all() and y[2, 1] > 1.7e38
    z = ref.quantised(np.array([[448.0, 17.0, 18.0, 19.0, 2.0 ** -9, 2.0 ** -10, -0.0146484375]]), "e4m3")[0]
    # 17 lies between 16 and 18 and 19 between 18 and 20; the last is 7.5 steps of 2^-9, and 8 is even
    assert z.tolist() == [448.0, 16.0, 18.0, 20.0, 2.0 ** -9, 0.0, -8 * 2.0 ** -9]
    for fmt in ("i8", "e4m3"):  # every code stands for itself
        v = ref.meaning(fmt)
        v = v[np.abs(v) <= ref.TOP[fmt]]
        row = np.concatenate([v, [ref.TOP[fmt]]])
        assert (ref.quantised(row, fmt)[:-1] == v).all()
