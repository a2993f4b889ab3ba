"""Calls of the score head that its documentation allows at the edges of what it says: rows without a class, odd tensors, other streams, empty
batches.  (test_score_head.py holds the operators against their formulas.)"""
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(scope="module")
def eng():
    import opal_amd
    e = opal_amd.Engine(0)
    yield e
    e.close()


@pytest.mark.gpu
@pytest.mark.parametrize("K", [1, 2, 10, 300, 2500, 9000])
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_class_one_when_nothing_is_above_minus_infinity(eng, t, K):
    """NaN never wins, and a class at -inf is ruled out: also where a NaN stands before it the answer is class 1."""
    inf, nan = float("inf"), float("nan")
    s = torch.full((6, K), -inf)
    s[1, 0] = nan
    s[2, : K // 2 + 1] = nan
    s[3] = nan
    s[4, K - 1] = nan
    s[5, 0] = nan
    s[5, K - 1] = torch.finfo(t).min           # the lowest number is above -inf
    cls, prob = eng.softmax_class(s.to(t).cuda())
    assert cls.tolist() == [1, 1, 1, 1, 1, K]
    prob = prob.cpu()
    assert prob[0] == 0 and prob[1:5].isnan().all()
    assert prob[5] == 1 if K == 1 else prob[5].isnan()


@pytest.mark.gpu
def test_a_flag_without_a_truth_value_raises_its_own_error(eng):
    class Neither:
        def __bool__(self):
            raise LookupError("neither")
    x, w = torch.randn(4, 8, device="cuda"), torch.randn(6, 8, device="cuda")
    one, labels = torch.ones(4, device="cuda"), torch.ones(4, dtype=torch.int32, device="cuda")
    for call in (lambda f: eng.layer_norm(x, want_stats=f), lambda f: eng.layer_norm_backward(x, x, None, one, one, want_dx=f),
                 lambda f: eng.layer_norm_backward(x, x, None, one, one, want_params=f), lambda f: eng.linear(x, w, want_pre=f),
                 lambda f: eng.linear_grad_weight(x, x, want_bias=f), lambda f: eng.softmax_loss(x, labels, want_grad=f)):
        with pytest.raises(LookupError, match="neither"):
            call(Neither())


def test_views_that_are_still_to_be_negated_are_refused():
    """The imaginary part of a conjugate is such a view: what lies in memory has the other sign."""
    from opal_amd._lib import bind
    b = bind()
    z = torch.complex(torch.randn(3, 4), torch.randn(3, 4)).conj()
    x = z.imag[:, :1]
    assert x.is_neg() and not x.resolve_neg().is_neg()
    for call in (lambda: b.softmax_class(0, 0, x), lambda: b.layer_norm(0, 0, x, None, None, 1e-5, None, False), lambda: b.linear_grad_weight(0, 0, x, x, True)):
        with pytest.raises(ValueError, match="resolve_neg"):
            call()


@pytest.mark.gpu
def test_vectors_that_are_still_to_be_negated_are_refused(eng):
    z = torch.complex(torch.randn(1), torch.randn(1)).cuda().conj()
    gamma = z.imag                             # one column: contiguous
    x = torch.randn(5, 1, device="cuda")
    with pytest.raises(ValueError, match="gamma.*resolve_neg"):
        eng.layer_norm(x, gamma)
    y, _, _ = eng.layer_norm(x, gamma.resolve_neg())
    assert y.shape == (5, 1)


def test_only_the_score_head_needs_its_extension_module(monkeypatch):
    """An Engine comes up, and is used, where the extension is absent or does not load; the first call that needs it says so.  (No GPU: the
    library and torch's streams are stand-ins.)"""
    import types
    import opal_amd.engine as engine

    def absent():
        raise ImportError("no extension here")
    library = types.SimpleNamespace(opal_ctx_create=lambda *a: 0, opal_ctx_destroy=lambda h: 0, opal_sync=lambda h: 0)
    monkeypatch.setattr(engine, "bind", absent)
    monkeypatch.setattr(engine, "lib", lambda: library)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "set_device", lambda d: None)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d: types.SimpleNamespace(cuda_stream=0))
    e = engine.Engine(0)
    e.sync()
    for call in (lambda: e.softmax_class(None), lambda: e.linear(None, None), lambda: e.layer_norm(None)):
        with pytest.raises(ImportError, match="no extension here"):
            call()
    e.close()


def test_a_stale_extension_module_is_noticed(monkeypatch):
    """Built from other sources, or for another torch, than those at hand: refused, as a library that lacks a symbol is."""
    from opal_amd import _lib
    module = _lib.bind()
    assert module.source == _lib.bind_source() and module.torch == torch.__version__
    with monkeypatch.context() as m:
        m.setattr(module, "torch", "1.0.0")
        with pytest.raises(ImportError, match="for torch 1.0.0"):
            _lib.bind()
    with monkeypatch.context() as m:
        m.setattr(_lib, "bind_source", lambda: "another")
        with pytest.raises(ImportError, match="stale"):
            _lib.bind()
    with monkeypatch.context() as m:                           # an installation without the sources
        m.setattr(_lib, "BIND_SOURCES", ("/nowhere/opal_bind.cpp",))
        assert _lib.bind_source() is None and _lib.bind() is module
    assert _lib.bind() is module


@pytest.mark.gpu
def test_a_workspace_is_not_handed_out_while_the_engine_works(eng):
    """With the engine on another stream than torch's current one: memory that a call gives back when it returns (its workspace) is not given to
    the current stream, which waits for the engine's only after that."""
    given = []

    def call(ctx, index, x):
        work = torch.empty(33 << 20, dtype=torch.uint8, device="cuda")           # a block of its own
        given.append(work.data_ptr())
        out = x + 1
        del work
        with torch.cuda.stream(side):                                            # as another thread would, between the call and the wait
            given.append(torch.empty(33 << 20, dtype=torch.uint8, device="cuda").data_ptr())
        return (out,)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    with torch.cuda.stream(side):
        x = torch.zeros(1000, device="cuda")
        out, = eng._run(call, (x,))
        assert given[0] != given[1]
        assert torch.equal(out, torch.ones(1000, device="cuda"))
    side.synchronize()


@pytest.mark.gpu
def test_refusals_on_another_stream_are_the_refusals(eng):
    """An argument that is no tensor, or is on the CPU, is refused as it is on the engine's stream; the streams stay in order."""
    x, w = torch.randn(4, 8, device="cuda"), torch.randn(6, 8, device="cuda")
    want = eng.linear(x, w)[0]
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()) as _:
        for call in (lambda: eng.linear(x, [1.0]), lambda: eng.linear(x.cpu(), w), lambda: eng.linear(x, None), lambda: eng.softmax_class(None)):
            with pytest.raises(ValueError):
                call()
        assert torch.equal(eng.linear(x, w)[0], want)


@pytest.mark.gpu
def test_results_on_another_stream_keep_their_memory_until_it_is_done(eng):
    """Results that are used on the current stream and dropped: the engine's next calls must not write over them first."""
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(4096, 700, device="cuda", generator=g).to(BF16)
    dy = torch.randn(4096, 512, device="cuda", generator=g).to(BF16)
    want = eng.linear_grad_weight(dy, x)
    torch.cuda.synchronize()
    side, heavy = torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
    with torch.cuda.stream(side):
        kept = []
        for i in range(6):
            dw, db = eng.linear_grad_weight(dy, x)
            for _ in range(3):
                heavy @ heavy                  # work ahead of the results' use
            kept.append((dw * 1.0, db * 1.0))
            del dw, db
            eng.linear_grad_weight(-dy, x)     # asks for memory of the same size at once
    side.synchronize()
    for dw, db in kept:
        assert torch.equal(dw, want[0]) and torch.equal(db, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("n", [3, 300])
def test_relu_and_nan(eng, t, n):
    """As the header says: NaN stays NaN, and neither it nor 0 passes a gradient on."""
    nan = float("nan")
    x = torch.randn(n, 24, device="cuda").to(t)
    w = torch.eye(24, device="cuda").to(t)
    x[1, 5], x[2] = nan, 0.0
    y, pre = eng.linear(x, w, activation="relu", want_pre=True)
    assert y[1].isnan().all() and not y[2].any() and torch.equal(y[0], x[0].clamp(min=0))         # (NaN times 0 is in each of the row's sums)
    pre = pre.clone()
    pre[1] = nan
    dx = eng.linear_grad_input(torch.ones(n, 24, device="cuda").to(t), w, pre=pre, activation="relu")
    assert not dx[1].any() and not dx[2].any() and torch.equal(dx[0], (x[0] > 0).to(t))


# ------------------------------------------------------------------------------ the head itself (opal_amd/head.py)
class HostEngine:
    """What ScoreHead needs of an engine to hold parameters: no GPU."""
    torch = torch
    device = torch.device("cpu")
    K = 5


def test_answers_of_no_fragments():
    from opal_amd.engine import DeviceBatch
    from opal_amd.head import ScoreHead, batch_scores
    head = ScoreHead(HostEngine, 5, 3)
    empty = DeviceBatch(torch.empty(0, dtype=torch.uint8), torch.zeros(1, dtype=torch.int64), torch.zeros(1, dtype=torch.int32), 0, 0)
    cls, prob = head.answers(empty, True)
    assert cls.shape == (0,) and cls.dtype == torch.int32 and prob.shape == (0,) and prob.dtype == F32
    assert list(batch_scores(HostEngine, empty, True)) == []


@pytest.mark.gpu
@pytest.mark.parametrize("n,K", [(1, 5), (700, 63), (3000, 356), (16384, 1563)])
def test_a_fresh_head_answers_as_the_linear_model(eng, n, K):
    """Also where the two highest scores are close: 2^-16 apart, which 16 bits cannot tell.  In 32 bits a score of less than 4, less its mean and
    scaled, is off by at most 4 (2^-24 + 2 2^-24) of the scale, twice that between two of them: 2^-18.4."""
    from opal_amd.head import ScoreHead
    g = torch.Generator().manual_seed(n + K)
    s = (torch.randn(n, K, generator=g) * 0.3 - 0.6).clamp(-1, 1)
    pair = torch.rand(n, K, generator=g).argsort(1)[:, :2]                       # two classes, the first of them a little above the other
    top = 1 + torch.rand(n, generator=g)
    s.scatter_(1, pair, torch.stack([top, top - 2.0 ** -16], 1))
    head = ScoreHead(eng, K, 16, seed=1)
    cls, prob = head.predict(s.cuda())
    assert torch.equal(cls.cpu().long() - 1, pair[:, 0])
    # the difference of two z is off by 24 U rstd (above) and by rstd's own error, (K + 8) U of it; the sum of K exponentials by (K + 8) U
    U, d = 2.0 ** -24, s.double()
    rstd = (d.var(1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    z = (d - d.mean(1, keepdim=True)) * rstd
    p = torch.softmax(z, 1).amax(1)
    tol = ((K + 8) * (1 + z.amax(1) - z.amin(1)) + 24 * rstd[:, 0]) * U
    assert ((prob.cpu().double() - p).abs() <= tol * p).all()


def test_a_head_knows_its_model(tmp_path):
    """A model of the same classes that was put in the place of the one the head was trained behind is noticed."""
    from opal_amd.head import ScoreHead, model_digest
    model, head_file = tmp_path / "m.model", str(tmp_path / "m.head")
    model.write_bytes(bytes(range(256)) * 40)
    ScoreHead(HostEngine, 5, 3, seed=2).save(head_file, model=str(model))
    assert ScoreHead.load(HostEngine, head_file, model=str(model)).K == 5 and ScoreHead.load(HostEngine, head_file).hidden == 3
    whole = model.read_bytes()
    assert model_digest(str(model), piece=100) != model_digest(str(model), piece=1 << 20)      # pieces count, and are 64 MiB
    for at in (0, 5000, len(whole) - 1):
        model.write_bytes(whole[:at] + bytes([whole[at] ^ 1]) + whole[at + 1:])
        with pytest.raises(RuntimeError, match="another model"):
            ScoreHead.load(HostEngine, head_file, model=str(model))
    for other in (whole[:-1], whole + b"x", b""):
        model.write_bytes(other)
        with pytest.raises(RuntimeError, match="another model"):
            ScoreHead.load(HostEngine, head_file, model=str(model))
    model.write_bytes(whole)
    assert torch.equal(ScoreHead.load(HostEngine, head_file, model=str(model)).params["w1"], ScoreHead(HostEngine, 5, 3, seed=2).params["w1"])
    raw = open(head_file, "rb").read()
    for bad in (raw[:-1], raw + b"x", raw[:8] + b"\x03" + raw[9:], raw[:8] + b"\x01" + raw[9:], raw[:30]):
        open(head_file, "wb").write(bad)
        with pytest.raises(RuntimeError):
            ScoreHead.load(HostEngine, head_file, model=str(model))
        with pytest.raises(RuntimeError):
            ScoreHead.read(head_file)
    ScoreHead(HostEngine, 5, 3).save(head_file)                                    # without a model: as it is
    assert ScoreHead.load(HostEngine, head_file, model=str(model)).K == 5


@pytest.mark.gpu
def test_predict_refuses_the_head_of_another_model(tmp_path):
    import argparse
    import numpy as np
    from opal_amd import model as model_io, opal
    from opal_amd.head import HEAD_FILE, ScoreHead
    rng = np.random.default_rng(3)
    K, bits = 5, 16
    for d in ("model", "test"):
        os.makedirs(tmp_path / d)
    with open(os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden", "patterns_k64_t16_m1_s7.txt")) as f:
        (tmp_path / "model" / "patterns.txt").write_text(f.read())
    (tmp_path / "model" / "vw-dico.txt").write_text("".join("tax%d\t%d\n" % (i, i) for i in range(1, K + 1)))
    (tmp_path / "test" / "reads.fasta").write_text("".join(">r%d\n%s\n" % (i, "".join(rng.choice(list("ACGT"), size=120))) for i in range(20)))
    model = str(tmp_path / "model" / "vw-model_final.model")
    weights = [(rng.standard_normal(1 << bits) * 0.05).astype(np.float32) for _ in range(2)]
    model_io.save_model(model, weights[0], K, bits)
    ScoreHead(HostEngine, K, 4, seed=1).save(str(tmp_path / "model" / HEAD_FILE), model=model)

    def predict(out, **more):
        opal.predict(str(tmp_path / "model"), str(tmp_path / "test"), str(tmp_path / out), argparse.Namespace(kmer=64, reverse_complement=True, **more))
        return (tmp_path / out / "test.fragments-db.preds.taxid").read_text().split()
    assert predict("a") == predict("b", no_head=True)                              # a fresh head: the linear model's answers
    model_io.save_model(model, weights[1], K, bits)
    with pytest.raises(RuntimeError, match="another model"):
        predict("c")
    assert len(predict("d", no_head=True)) == 20


@pytest.mark.gpu
def test_answers_on_another_stream_wait_for_the_fragments(eng):
    """Fragments that the current stream is still bringing when it asks for their scores or answers; the engine runs on another one."""
    import numpy as np
    import opal_amd
    from opal_amd.engine import DeviceBatch
    from opal_amd.head import ScoreHead, batch_scores
    rng = np.random.default_rng(11)
    K, bits, n = 24, 16, 500
    e = opal_amd.Engine(0)
    e.set_patterns(np.array([range(8), range(0, 16, 2)], dtype=np.int32), 16)
    e.load_weights((rng.standard_normal(1 << bits) * 0.1).astype(np.float32), K, bits)
    e.set_vw_options()
    text = "".join(">r%d\n%s\n" % (i, "".join(rng.choice(list("ACGT"), size=100))) for i in range(n))
    batch = e.ingest_fasta(np.frombuffer(text.encode(), dtype=np.uint8).copy())
    head = ScoreHead(e, K, 16, seed=5)
    want = head.answers(batch, True, rows=512)
    scores = torch.cat([s for _, s in batch_scores(e, batch, True, limit=4 * K * 200)])
    none = head.answers(DeviceBatch(torch.zeros_like(batch.data), batch.off, batch.len, n, batch.nbytes), True, rows=512)
    assert not torch.equal(none[0], want[0])
    torch.cuda.synchronize()
    side, heavy = torch.cuda.Stream(), torch.randn(8192, 8192, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for ask in (lambda b: head.answers(b, True, rows=512), lambda b: (torch.cat([s for _, s in batch_scores(e, b, True, limit=4 * K * 200)]),)):
            late = DeviceBatch(torch.zeros_like(batch.data), batch.off, batch.len, n, batch.nbytes)
            for _ in range(10):
                heavy @ heavy
            late.data.copy_(batch.data)
            got = [x.clone() for x in ask(late)]
            late.data.zero_()                  # behind the answers
            side.synchronize()
            for a, b in zip(got, want if len(got) == 2 else (scores,)):
                assert torch.equal(a, b)
    e.close()
