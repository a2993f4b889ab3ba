"""The score head's matrix products by the kernel that makes them: which one a size reaches is asked of the rules themselves (a small
host program, no GPU), so that a change of rule cannot move what these tests cover.  Tolerances as in test_score_head.py."""
import os
import subprocess
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch  # noqa: E402

from test_score_head import act64, close, rounding, slope64, U  # noqa: E402

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


# ------------------------------------------------------------------------------ every kernel against the formula
ACTS = ["none", "relu", "silu", "gelu"]


def forward_case(t, n, k, m, large):
    return "product %d %d %d %d %d %d %d 1" % (FWD, CODE[t], n, m, k, CUS, large)


def input_case(t, n, k, m, large):
    return "product %d %d %d %d %d %d %d 1" % (GIN, CODE[t], n, k, m, CUS, large)


# n, k, m: forward [n, k] x [m, k]; input gradient [n, m] x [m, k]
BIG_FORWARD = [(33000, 1027, 501), (66000, 270, 1000)]         # 256 x 256: a last round that goes to smaller tiles, sums that end inside a chunk, cut columns
PAIR_FORWARD = [(16400, 192, 511), (8200, 355, 1030), (70001, 33, 257)]
BIG_INPUT = [(33000, 1027, 501), (17000, 1000, 71)]
MIDDLE_ODD = [(9001, 1563, 1041)]                              # rows that do not begin on 16 bytes


def test_the_sizes_below_reach_the_kernels_they_are_for(rules):
    for t in (F16, BF16):
        for shape in BIG_FORWARD:
            assert rules([forward_case(t, *shape, 1)]) == [[BIG]], shape
        for shape in PAIR_FORWARD:
            assert rules([forward_case(t, *shape, 1)]) == [[PAIR]], shape
        for shape in BIG_INPUT:
            assert rules([input_case(t, *shape, 1)]) == [[BIG]], shape
        for n, k, m in MIDDLE_ODD:
            assert rules([forward_case(t, n, k, m, 0), input_case(t, n, k, m, 0)]) == [[MIDDLE], [MIDDLE]]
            assert rules(["weight %d %d %d %d" % (n, k, m, CODE[t])])[0][0] == BIG         # whose splits the 128 x 128 tiles take there
    for n, k, m in WEIGHT32:
        assert rules(["weight %d %d %d 0" % (n, k, m)])[0][0] == MIDDLE


def test_weight_gradients_in_32_bits_take_128_tiles_where_those_were_faster(rules):
    for n, k, m, tile in ((100000, 1564, 512, MIDDLE), (6000, 1564, 512, MIDDLE), (4096, 1564, 512, MIDDLE), (16384, 356, 512, MIDDLE), (100000, 200, 1000, MIDDLE),
                          (6000, 356, 512, SMALL), (3000, 520, 400, SMALL), (4096, 356, 512, SMALL), (50000, 130, 1564, SMALL), (100000, 63, 64, SMALL)):
        assert rules(["weight %d %d %d 0" % (n, k, m)])[0][0] == tile, (n, k, m)


def random(g, t):
    """rnd(rows, cols, scale, rows on 16 bytes): a matrix whose gaps are NaN"""
    def rnd(a, b, scale=1.0, aligned=True, t=t):
        step = 16 // torch.empty(0, dtype=t).element_size()
        full = torch.full((a, -(-b // step) * step if aligned else b), float("nan"), device="cuda", dtype=t)
        full[:, :b] = (torch.randn(a, b, device="cuda", generator=g) * scale).to(t)
        return full[:, :b]
    return rnd


def some_rows(n):
    """the first and the last rows, where a last round's smaller tiles begin and end, and some between"""
    return torch.cat([torch.arange(200), torch.randint(0, n, (300,), generator=torch.Generator().manual_seed(n)), torch.arange(n - 400, n)])


def check_forward(eng, rnd, t, n, k, m, act, res, out, aligned=True):
    x, w, bias = rnd(n, k, 1.0, aligned), rnd(m, k, k ** -0.5, aligned), rnd(1, m, 1.0, True, F32)[0].clone()
    r = rnd(n, m, 1.0, aligned, res) if res is not None else None
    y, pre = eng.linear(x, w, bias, activation=act, residual=r, out_dtype=out, want_pre=True)
    at = some_rows(n)
    x64, w64, b64 = x[at.cuda()].double().cpu(), w.double().cpu(), bias.double().cpu()
    p = x64 @ w64.t() + b64
    dp = (k + 3) * U * (x64.abs() @ w64.abs().t() + b64.abs())
    close(pre[at.cuda()], p, dp + rounding(p.abs() + dp, t), "pre")
    a = act64(p, act)
    # the largest slope is 1.13; the exponential, the reciprocal and their argument cost a few U of the value and |argument| U of the sigmoid
    da = 1.13 * dp + U * (8 + 4 * p.abs() + 2 * p.abs() ** 3) * a.abs() + 1e-37
    ref = a + (r[at.cuda()].double().cpu() if r is not None else 0.0)
    d = da + U * (ref.abs() + a.abs() + da)
    close(y[at.cuda()], ref, d + rounding(ref.abs() + d, out), "y")
    assert torch.isfinite(y.float()).all() and torch.isfinite(pre.float()).all()


def check_input(eng, rnd, t, n, k, m, act, res, out, aligned=True):
    dy, w, pre = rnd(n, m, 0.1, aligned), rnd(m, k, k ** -0.5, aligned), rnd(n, k, 1.0, aligned)
    r = rnd(n, k, 1.0, aligned, res) if res is not None else None
    dx = eng.linear_grad_input(dy, w, pre=pre if act != "none" else None, activation=act, residual=r, out_dtype=out)
    at = some_rows(n)
    dy64, w64, pre64 = dy[at.cuda()].double().cpu(), w.double().cpu(), pre[at.cuda()].double().cpu()
    s, p = slope64(pre64, act), dy64 @ w64
    d = s.abs() * (m + 2) * U * (dy64.abs() @ w64.abs())
    ds = U * (16 + 16 * pre64.abs() + 8 * pre64.abs() ** 3) if act in ("silu", "gelu") else 0.0
    ref = p * s + (r[at.cuda()].double().cpu() if r is not None else 0.0)
    d = d + p.abs() * ds + 2 * U * (ref.abs() + (p * s).abs())
    close(dx[at.cuda()], ref, d + rounding(ref.abs() + d, out), "dx")
    assert torch.isfinite(dx.float()).all()


def check_weight(eng, rnd, n, k, m, aligned=True):
    dy, x = rnd(n, m, 0.1, aligned), rnd(n, k, 1.0, aligned)
    dw, db = eng.linear_grad_weight(dy, x)
    dy64, x64 = dy.double().cpu(), x.double().cpu()
    close(dw, dy64.t() @ x64, (n + 2) * U * (dy64.abs().t() @ x64.abs()) + 1e-38, "dw")
    close(db, dy64.sum(0), (n + 2) * U * dy64.abs().sum(0) + 1e-38, "db")


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("res", ["without", "own", F32])
@pytest.mark.parametrize("out", ["own", F32])
@pytest.mark.parametrize("n,k,m", BIG_FORWARD + PAIR_FORWARD)
def test_large_forward_epilogues(eng, t, act, res, out, n, k, m):
    g = torch.Generator(device="cuda").manual_seed(n + k + m)
    pick = {"without": None, "own": t, F32: F32}
    check_forward(eng, random(g, t), t, n, k, m, act, pick[res], pick[out])


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("res", ["without", "own", F32])
@pytest.mark.parametrize("out", ["own", F32])
@pytest.mark.parametrize("n,k,m", BIG_INPUT)
def test_large_input_gradient_epilogues(eng, t, act, res, out, n, k, m):
    g = torch.Generator(device="cuda").manual_seed(n + k + m)
    pick = {"without": None, "own": t, F32: F32}
    check_input(eng, random(g, t), t, n, k, m, act, pick[res], pick[out])


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("n,k,m", MIDDLE_ODD)
def test_large_products_of_rows_that_do_not_begin_on_16_bytes(eng, t, n, k, m):
    """Contiguous matrices of odd width: 128 x 128 tiles by way of registers, in all three directions."""
    g = torch.Generator(device="cuda").manual_seed(n + k + m)
    for act, res, out in (("gelu", t, F32), ("silu", None, t)):
        check_forward(eng, random(g, t), t, n, k, m, act, res, out, aligned=False)
        check_input(eng, random(g, t), t, n, k, m, act, res, out, aligned=False)
    check_weight(eng, random(g, t), n, k, m, aligned=False)


WEIGHT32 = [(12033, 511, 397), (6010, 1564, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,k,m", WEIGHT32)
@pytest.mark.parametrize("aligned", [True, False])
def test_weight_gradient_in_32_bits_with_128_tiles(eng, n, k, m, aligned):
    g = torch.Generator(device="cuda").manual_seed(n + k + m)
    rnd = random(g, F32)
    if not aligned and k % 4 == 0:                             # an even width: one element between the rows
        wide = lambda a, b, scale=1.0, aligned=True: rnd(a, b + 1, scale, False)[:, :b]  # noqa: E731
        check_weight(eng, wide, n, k, m)
    else:
        check_weight(eng, rnd, n, k, m, aligned)
