"""The score head's matrix products by the kernel that makes them: which one a size reaches is asked of the rules themselves (a small
host program, no GPU), so that a change of rule cannot move what these tests cover.  Tolerances as in test_score_head.py."""
import os
import subprocess
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
CODE = {F32: 0, F16: 1, BF16: 2}
FWD, GIN = 0, 1
CUS = 256                                      # of the card
SMALL, MIDDLE, BIG, FEW, PAIR, FEW_WEIGHT = 0, 1, 2, 3, 4, 5


@pytest.fixture(scope="session")
def rules(tmp_path_factory):
    """rules(lines): the answers of opal_linear_rules.h, lists of integers."""
    exe = str(tmp_path_factory.mktemp("rules") / "rules")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-I%s/include" % ROOT, "-I%s/opal_amd/csrc" % ROOT, "%s/tests/native/linear_rules.cpp" % ROOT, "-o", exe])

    def ask(lines):
        run = subprocess.run([exe], input="\n".join(lines) + "\n", capture_output=True, text=True, timeout=60, check=True)
        got = [[int(x) for x in line.split()] for line in run.stdout.splitlines()]
        assert len(got) == len(lines)
        return got
    return ask


@pytest.fixture(scope="module")
def eng():
    import opal_amd
    e = opal_amd.Engine(0)
    yield e
    e.close()


# ------------------------------------------------------------------------------ no rows
def test_a_sum_over_no_rows_never_takes_the_kernel_that_asks_ahead(rules):
    """The 256 x 256 kernel asks for the chunks of its first steps before it looks at their number: a weight gradient over no rows is another's."""
    sizes = [(1, 1), (5, 7), (129, 129), (512, 1564), (8192, 16384), (11776, 11776), (1 << 20, 1 << 10), (1 << 20, 1 << 20)]
    asked = [(i, o, t) for i, o in sizes + [(b, a) for a, b in sizes] for t in CODE.values()]
    for (i, o, t), (tile, splits, _) in zip(asked, rules(["weight 0 %d %d %d" % a for a in asked])):
        assert tile != BIG and splits == 1, (i, o, t)
    assert rules(["weight 1 8192 16384 2", "weight 100000 512 1564 2"]) == [[BIG, 1, 64], [BIG, 18, 5568]]       # and with rows it is that one's


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F16, BF16, F32])
def test_weight_gradient_over_no_rows(eng, t):
    """Zeros, at sizes that take the largest tiles as soon as there is a row; nothing behind the matrix is written."""
    from opal_amd._lib import check
    k, m = 8192, 16384
    dw, db = torch.full((m + 1, k), float("nan"), device="cuda"), torch.full((m + 1,), float("nan"), device="cuda")
    assert eng._lib.opal_linear_grad_weight_workspace(0, k, m, CODE[t]) == 0
    check(eng._lib.opal_linear_grad_weight(eng._h, None, m, None, k, CODE[t], 0, k, m, dw.data_ptr(), k, db.data_ptr(), None, 0), eng._h)
    assert not dw[:m].any() and dw[m].isnan().all() and not db[:m].any() and db[m].isnan()
    dw, db = eng.linear_grad_weight(torch.empty(0, m, dtype=t, device="cuda"), torch.empty(0, k, dtype=t, device="cuda"))
    assert dw.shape == (m, k) and not dw.any() and not db.any()
