"""The score head as `train --head` makes it and `predict` uses it (opal_amd/head.py)."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch  # noqa: E402

from opal_amd import head as head_mod  # noqa: E402
from opal_amd import opal  # noqa: E402
from opal_amd.head import HEAD_FILE, ScoreHead, batch_scores  # noqa: E402


class HostEngine:
    """What ScoreHead needs of an engine to hold parameters: no GPU."""
    torch = torch
    device = torch.device("cpu")


@pytest.fixture(scope="module")
def eng():
    import opal_amd
    e = opal_amd.Engine(0)
    yield e
    e.close()


def test_file_round_trip(tmp_path):
    h = ScoreHead(HostEngine, 13, 5, seed=3)
    g = torch.Generator().manual_seed(1)
    for p in h.params.values():
        p.copy_(torch.randn(p.shape, generator=g))
    path = str(tmp_path / HEAD_FILE)
    h.save(path)
    back = ScoreHead.load(HostEngine, path)
    assert (back.K, back.hidden) == (13, 5)
    for n, p in h.params.items():
        assert torch.equal(back.params[n], p), n
    for n in ("w1", "w2"):
        assert torch.equal(back._half[n], h.params[n].to(torch.bfloat16)) and back._half[n].stride(0) % 8 == 0


def test_a_fresh_head_is_the_linear_model_and_the_same_for_a_seed():
    a, b, c = ScoreHead(HostEngine, 7, 9, seed=1), ScoreHead(HostEngine, 7, 9, seed=1), ScoreHead(HostEngine, 7, 9, seed=2)
    assert torch.equal(a.params["w1"], b.params["w1"]) and not torch.equal(a.params["w1"], c.params["w1"])
    assert not a.params["w2"].any() and not a.params["b2"].any()


@pytest.mark.parametrize("damage", ["magic", "short", "long", "version", "empty", "size"])
def test_other_files_are_refused(tmp_path, damage):
    path = str(tmp_path / HEAD_FILE)
    ScoreHead(HostEngine, 4, 3).save(path)
    raw = bytearray(open(path, "rb").read())
    if damage == "magic":
        raw[0] ^= 1
    elif damage == "short":
        raw = raw[:-1]
    elif damage == "long":
        raw += b"x"
    elif damage == "version":
        raw[8] = 2
    elif damage == "empty":
        raw = b""
    else:
        raw[12:16] = b"\xff\xff\xff\xff"
    open(path, "wb").write(bytes(raw))
    with pytest.raises(RuntimeError):
        ScoreHead.read(path)


def test_sizes_are_checked():
    for K, H in ((0, 4), (4, 0), (1 << 21, 4), (4, 1 << 21)):
        with pytest.raises(ValueError):
            ScoreHead(HostEngine, K, H)


def test_flags():
    p = opal.build_parser()
    a = p.parse_args(["train", "a", "b"])
    assert a.head == 0
    a = p.parse_args(["simulate", "a", "b", "c", "--head", "64", "--head-batches", "3", "--head-rows", "128", "--head-rate", "0.1"])
    assert (a.head, a.head_batches, a.head_rows, a.head_rate) == (64, 3, 128, 0.1)
    a = p.parse_args(["predict", "a", "b", "c", "--no-head", "--probabilities"])
    assert a.no_head and a.probabilities
    opal.check_head_options(1, 1, 1, 0.1)
    for bad in ((-1, 1, 1, 0.1), (1 << 21, 1, 1, 0.1), (4, 0, 1, 0.1), (4, 1, 0, 0.1), (4, 1, 1, 0.0), (4, 1, 1, float("nan"))):
        with pytest.raises(ValueError):
            opal.check_head_options(*bad)


@pytest.mark.gpu
@pytest.mark.parametrize("n,K,H", [(1, 2, 1), (40, 6, 9), (257, 63, 64)])
def test_gradients_and_step(eng, n, K, H):
    """The head's gradients are those of its operators (test_score_head.py holds them against the formula and differences), and a
    step moves every parameter by AdaGrad's rule: rate * g / sqrt(sum of g^2)."""
    import test_score_head as ops
    s, labels, gamma, beta, w1, b1, w2, b2 = (x.cuda() for x in ops.head_inputs(n, K, H, ops.BF16))
    head = ScoreHead(eng, K, H, params={k: v.float().cpu().numpy() for k, v in zip(head_mod._NAMES, (gamma, beta, w1, b1, w2, b2))})
    loss, g = head.gradients(s, labels)
    want = ops.head_step(eng, s, labels, gamma, beta, head._half["w1"], b1, head._half["w2"], b2, ops.BF16, 1.0 / n)
    assert torch.equal(loss, want[0])
    for name, ref in zip(head_mod._NAMES, want[2:]):
        assert torch.equal(g[name], ref), name
    before = {k: v.clone() for k, v in head.params.items()}
    head.train_step(s, labels, rate=0.25)
    for name, p in head.params.items():
        assert torch.equal(head.grads2[name], g[name] * g[name]), name
        step = 0.25 * g[name].double() / (g[name].double().abs() + 1e-8)
        # the root of a float32 square is exact to a few roundings, but a square below 2^-126 has fewer digits: such gradients are set aside
        ok = g[name].abs() > 2.0 ** -62
        off = (p.double() - (before[name].double() - step)).abs()
        assert (off[ok] <= 2.0 ** -21 * 0.25 + 2.0 ** -24 * before[name].double().abs()[ok]).all(), name
        assert (off <= 0.26 + 2.0 ** -24 * before[name].double().abs()).all(), name
    for name in ("w1", "w2"):
        assert torch.equal(head._half[name], head.params[name].to(torch.bfloat16))


@pytest.mark.gpu
def test_scores_in_parts_are_the_batch(eng):
    rng = np.random.default_rng(5)
    K, bits = 6, 16
    eng.set_patterns(np.array([range(8), range(0, 16, 2)], dtype=np.int32), 16)
    eng.load_weights(rng.standard_normal(1 << bits).astype(np.float32), K, bits)
    eng.set_vw_options()
    text = "".join(">r%d\n%s\n" % (i, "".join(rng.choice(list("ACGT"), size=20 + i % 7))) for i in range(101))
    batch = eng.ingest_fasta(np.frombuffer(text.encode(), dtype=np.uint8).copy())
    whole = eng.predict(batch, True, want_scores=True)[1].clone()
    parts = list(batch_scores(eng, batch, True, limit=4 * K * 17))
    assert [lo for lo, _ in parts] == list(range(0, 101, 17))
    assert torch.equal(torch.cat([s for _, s in parts]), whole)
    assert [s.shape[0] for _, s in batch_scores(eng, batch, True, limit=1)] == [1] * 101


@pytest.mark.gpu
def test_cli_train_and_predict_with_a_head(tmp_path, capsys):
    rng = np.random.default_rng(12)
    K = 5
    genomes = ["".join(rng.choice(list("ACGT"), size=6000)) for _ in range(K)]
    for d in ("train", "test"):
        os.makedirs(tmp_path / d)
        with open(tmp_path / d / "A1.fasta", "w") as f:
            f.write("".join(">g%d\n%s\n" % (i, g) for i, g in enumerate(genomes)))
        with open(tmp_path / d / "A1.taxid", "w") as f:
            f.write("".join("%d\n" % (100 + i) for i in range(K)))
    common = ["-r", "-l", "200", "-c", "3", "--num-hash", "1", "--bits", "22"]

    def train(name, *more):
        np.random.seed(4)
        opal.main(["train", str(tmp_path / "train"), str(tmp_path / name)] + common + list(more))
        return open(tmp_path / name / "vw-model_final.model", "rb").read()
    plain = train("plain")
    headed = train("headed", "--head", "24", "--head-batches", "2", "--head-rows", "64")
    again = train("again", "--head", "24", "--head-batches", "2", "--head-rows", "64")
    assert plain == headed == again                                   # the linear model does not know of the head
    read = lambda *p: open(tmp_path.joinpath(*p), "rb").read()  # noqa: E731
    assert read("headed", HEAD_FILE) == read("again", HEAD_FILE) and not (tmp_path / "plain" / HEAD_FILE).exists()
    assert ScoreHead.read(str(tmp_path / "headed" / HEAD_FILE))[:2] == (K, 24)
    assert "head batch 1: " in read("headed", "vw-model_vwps.log").decode()

    def predict(model, out, *more):
        opal.main(["predict", str(tmp_path / model), str(tmp_path / "test"), str(tmp_path / out), "-r"] + list(more))
        return read(out, "test.fragments-db.preds.taxid").decode().split()
    with_head = predict("headed", "p_head", "--probabilities")
    prob = [float(x) for x in read("p_head", "test.fragments-db.preds.prob").decode().split()]
    assert len(with_head) == len(prob) == K and all(0 < x <= 1 for x in prob) and set(with_head) <= {str(100 + i) for i in range(K)}
    assert "score head: 24 hidden units" in read("p_head", "test.fragments-db_vwps.log").decode()
    assert predict("headed", "p_linear", "--no-head") == predict("plain", "p_plain")
    assert read("p_linear", "test.fragments-db.preds.vw") == read("p_plain", "test.fragments-db.preds.vw")
    # the answers are the head's own on the scores
    import opal_amd
    from opal_amd import model as model_io
    e = opal_amd.Engine(0)
    with open(tmp_path / "headed" / "patterns.txt") as f:
        e.set_patterns(opal_amd.parse_patterns(f.readlines(), 64), 64)
    model_io.load_model(str(tmp_path / "headed" / "vw-model_final.model"), e)
    batch = e.ingest_fasta(np.fromfile(tmp_path / "test" / "A1.fasta", dtype=np.uint8))
    head = ScoreHead.load(e, str(tmp_path / "headed" / HEAD_FILE))
    cls, p = head.answers(batch, True)
    scores = torch.zeros(16384, K, device="cuda")
    scores[:batch.n] = e.predict(batch, True, want_scores=True)[1]
    direct, q = head.predict(scores)
    assert torch.equal(cls, direct[:batch.n]) and torch.equal(p, q[:batch.n])
    assert [int(float(x.split()[0])) for x in read("p_head", "test.fragments-db.preds.vw").decode().splitlines()] == cls.tolist()
    assert ["%.6f" % x for x in p.tolist()] == read("p_head", "test.fragments-db.preds.prob").decode().split()
    e.close()
    # without the flag the older file of probabilities goes; without a head it is refused
    predict("headed", "p_head")
    assert not (tmp_path / "p_head" / "test.fragments-db.preds.prob").exists()
    with pytest.raises(ValueError, match="score head"):
        predict("plain", "p_plain", "--probabilities")
    # a new model without a head takes the old one's head away; several passes use the saved regressor
    assert train("again", "--num-passes", "2", "--head", "8") == train("plain", "--num-passes", "2")
    assert ScoreHead.read(str(tmp_path / "again" / HEAD_FILE))[:2] == (K, 8)
    train("again")
    assert not (tmp_path / "again" / HEAD_FILE).exists()
    with pytest.raises(ValueError, match="--head-rows"):
        train("again", "--head", "8", "--head-rows", "0")


def _predict_rank(rank, world, port, model_dir, test_dir, out_dir):
    import argparse
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank))
    opal.predict(model_dir, test_dir, out_dir, argparse.Namespace(kmer=64, reverse_complement=True, probabilities=True), chunk_bytes=10_000)


@pytest.mark.gpu
def test_answers_do_not_depend_on_pieces_or_ranks(tmp_path):
    """A file at once, in pieces, and dealt to two ranks (both on this GPU): the same classes and probabilities, byte for byte."""
    import argparse
    import socket
    import torch.multiprocessing as mp
    import opal_amd
    from opal_amd import model as model_io
    rng = np.random.default_rng(29)
    K, bits, H = 70, 18, 40
    for d in ("model", "test"):
        os.makedirs(tmp_path / d)
    with open(os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden", "patterns_k64_t16_m1_s7.txt")) as f:
        (tmp_path / "model" / "patterns.txt").write_text(f.read())
    (tmp_path / "model" / "vw-dico.txt").write_text("".join("tax%d\t%d\n" % (i, i) for i in range(1, K + 1)))
    model_io.save_model(str(tmp_path / "model" / "vw-model_final.model"), (rng.standard_normal(1 << bits) * 0.05).astype(np.float32), K, bits)
    params = dict(gamma=1 + 0.1 * rng.standard_normal(K), beta=0.1 * rng.standard_normal(K), w1=rng.standard_normal((H, K)) / 8, b1=rng.standard_normal(H) * 0.1,
                  w2=rng.standard_normal((K, H)) / 6, b2=rng.standard_normal(K) * 0.1)
    ScoreHead(HostEngine, K, H, params=params).save(str(tmp_path / "model" / HEAD_FILE))
    with open(tmp_path / "test" / "reads.fasta", "w") as f:
        for i in range(701):
            f.write(">r%d\n%s\n" % (i, "".join(rng.choice(list("ACGT"), size=int(rng.integers(40, 300))))))
    args = argparse.Namespace(kmer=64, reverse_complement=True, probabilities=True)
    opal.predict(str(tmp_path / "model"), str(tmp_path / "test"), str(tmp_path / "one"), args)
    opal.predict(str(tmp_path / "model"), str(tmp_path / "test"), str(tmp_path / "pieces"), args, chunk_bytes=10_000)
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    mp.spawn(_predict_rank, args=(2, port, str(tmp_path / "model"), str(tmp_path / "test"), str(tmp_path / "two")), nprocs=2, join=True)
    for name in ("test.fragments-db.preds.vw", "test.fragments-db.preds.taxid", "test.fragments-db.preds.prob"):
        a = (tmp_path / "one" / name).read_bytes()
        assert a.count(b"\n") == 701 and (tmp_path / "pieces" / name).read_bytes() == a and (tmp_path / "two" / name).read_bytes() == a
    e = opal_amd.Engine(0)
    with open(tmp_path / "model" / "patterns.txt") as f:
        e.set_patterns(opal_amd.parse_patterns(f.readlines(), 64), 64)
    model_io.load_model(str(tmp_path / "model" / "vw-model_final.model"), e)
    head = ScoreHead.load(e, str(tmp_path / "model" / HEAD_FILE))
    batch = e.ingest_fasta(np.fromfile(tmp_path / "test" / "reads.fasta", dtype=np.uint8))
    cls, prob = head.answers(batch, True)
    assert len(set(cls.tolist())) > 5
    few = head.answers(batch, True, rows=100)                      # parts that do not divide the batch: the first is these rows alone
    scores = e.predict(batch, True, want_scores=True)[1]
    for lo in (0, 100):
        part = head.predict(scores[lo:lo + 100].contiguous())
        assert torch.equal(few[0][lo:lo + 100], part[0]) and torch.equal(few[1][lo:lo + 100], part[1])
    assert few[0].shape == cls.shape and few[1].shape == prob.shape
    e.close()
