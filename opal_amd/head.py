"""The score head: a trained layer behind the linear model's per-class scores (`train --head H`, `predict`).

The linear model is K independent regressors: its scores are no probabilities and nothing corrects a class that is regularly taken
for a sister species.  (On reads of strains that neither has seen the head has not made the answers better, 0.9954 against 0.9972 of 64 species: what it
gives is a probability that orders them.)  The head reads all K scores s of a fragment,

    z = layer norm(s),   logits = z + W2 gelu(W1 z + b1) + b2,   p = softmax(logits),

and is trained by cross entropy on fragments the linear model has scored, with AdaGrad as the linear learner uses.  It starts as the
linear model itself (W2 = 0): the answers are the linear model's, up to scores that 32 bits of z cannot tell apart.  The work is
Engine.layer_norm, linear, linear_grad_input, linear_grad_weight, softmax_loss and softmax_class (hand-written HIP kernels); torch holds the parameters and makes the parameter update, a few passes over them.
No counterpart in the reference, whose answer is the argmax of the scores (opal.py:449-469)."""
import hashlib
import os
import struct
from concurrent.futures import ThreadPoolExecutor

import numpy as np

__all__ = ["ScoreHead", "HEAD_FILE", "batch_scores", "model_digest"]

HEAD_FILE = "vw-model_final.head"        # next to vw-model_final.model
_HDR = struct.Struct("<8sIII")           # magic, version, K, hidden; version 2: model_digest; then float32 gamma, beta, w1, b1, w2, b2
_DIGEST = 32                             # bytes
_MAGIC = b"OPALHEAD"
_NAMES = ("gamma", "beta", "w1", "b1", "w2", "b2")
EPS = 1e-5


def model_digest(path, piece=1 << 26):
    """What tells a linear model's file from another: sha256 of the sha256 of its pieces (of 64 MiB, side by side)."""
    def part(at):
        with open(path, "rb") as f:
            f.seek(at)
            return hashlib.sha256(f.read(piece)).digest()
    with ThreadPoolExecutor(min(8, os.cpu_count() or 1)) as pool:
        return hashlib.sha256(b"".join(pool.map(part, range(0, os.path.getsize(path), piece)))).digest()


def batch_scores(engine, batch, reverse, limit=1 << 30):
    """(first row, scores float32 [rows, K]) of a device batch of fragments, in parts of at most `limit` bytes (one row at least)."""
    from .engine import DeviceBatch
    rows = max(1, limit // (4 * engine.K))
    for lo in range(0, batch.n, rows):
        hi = min(batch.n, lo + rows)
        part = DeviceBatch(batch.data, batch.off[lo:hi], batch.len[lo:hi], hi - lo, batch.nbytes)
        with engine._own_stream(inputs=(part.data, part.off, part.len)) as results:
            scores = engine.predict(part, reverse, want_scores=True)[1]
            results.append(scores)
        yield lo, scores


class ScoreHead:
    def __init__(self, engine, K, hidden, seed=0, params=None):
        """params: dict of float32 numpy arrays (as load() reads them); else a fresh head of that seed."""
        t = engine.torch
        if not (1 <= K <= 1 << 20 and 1 <= hidden <= 1 << 20):
            raise ValueError("the head needs 1 .. 2^20 classes and hidden units")
        self.engine, self.K, self.hidden = engine, K, hidden
        if params is None:
            w1 = np.random.default_rng(seed).standard_normal((hidden, K), dtype=np.float32) / np.float32(np.sqrt(K))
            params = dict(gamma=np.ones(K), beta=np.zeros(K), w1=w1, b1=np.zeros(hidden), w2=np.zeros((K, hidden)), b2=np.zeros(K))
        self.params = {n: t.from_numpy(np.ascontiguousarray(params[n], dtype=np.float32)).to(engine.device) for n in _NAMES}
        self.grads2 = {n: t.zeros_like(p) for n, p in self.params.items()}             # AdaGrad's sums of squares
        self._half = {}
        for n in ("w1", "w2"):                                                         # what the products take: bfloat16, rows on 16 bytes
            r, c = self.params[n].shape
            self._half[n] = t.empty_strided((r, c), ((c + 7) & ~7, 1), dtype=t.bfloat16, device=engine.device)
        self._copy_weights()

    def _copy_weights(self):
        for n, h in self._half.items():
            h.copy_(self.params[n])

    def forward(self, scores, for_training=False):
        """logits float32 [n, K] (and what backward needs) of scores float32 [n, K].  An answer hangs on which of two close scores is the
        higher one: there the z that is added to the product stays in 32 bits.  A training step adds the bfloat16 z that the product
        takes, a pass over the scores less: its gradients are rounded to bfloat16 anyway."""
        e, t, p = self.engine, self.engine.torch, self.params
        z, mean, rstd = e.layer_norm(scores, p["gamma"], p["beta"], eps=EPS, out_dtype=t.bfloat16, want_stats=for_training)
        h, pre = e.linear(z, self._half["w1"], p["b1"], activation="gelu", want_pre=for_training)
        added = z if for_training else e.layer_norm(scores, p["gamma"], p["beta"], eps=EPS, out_dtype=t.float32)[0]
        logits, _ = e.linear(h, self._half["w2"], p["b2"], residual=added, out_dtype=t.float32)
        return (logits, (scores, z, mean, rstd, h, pre)) if for_training else logits

    def gradients(self, scores, labels):
        """(loss float32 [n], dict of the parameters' gradients of the mean loss over the labelled rows' share of n)."""
        e, t, p = self.engine, self.engine.torch, self.params
        logits, (scores, z, mean, rstd, h, pre) = self.forward(scores, for_training=True)
        loss, dl = e.softmax_loss(logits, labels, scale=1.0 / max(scores.shape[0], 1), out_dtype=t.bfloat16)
        g = {}
        g["w2"], g["b2"] = e.linear_grad_weight(dl, h)
        dpre = e.linear_grad_input(dl, self._half["w2"], pre=pre, activation="gelu")
        g["w1"], g["b1"] = e.linear_grad_weight(dpre, z)
        dz = e.linear_grad_input(dpre, self._half["w1"], residual=dl)
        _, g["gamma"], g["beta"] = e.layer_norm_backward(dz, scores, p["gamma"], mean, rstd, want_dx=False)
        return loss, g

    def train_step(self, scores, labels, rate=0.05):
        """One AdaGrad step on a batch; labels int32 [n], class ids 1..K (0: no known class).  Returns the loss per row."""
        loss, g = self.gradients(scores, labels)
        for n, p in self.params.items():
            s = self.grads2[n].addcmul_(g[n], g[n])
            p.addcdiv_(g[n], s.sqrt().add_(1e-8), value=-rate)
        self._copy_weights()
        return loss

    def predict(self, scores):
        """(class int32 [n], 1-based, its probability float32 [n])."""
        return self.engine.softmax_class(self.forward(scores))

    def answers(self, batch, reverse, rows=16384, limit=1 << 30):
        """predict() of a device batch of fragments.  Always as many rows at a time, the last ones filled up with zeros: another number of
        rows can choose another product kernel, whose sums have another order, and a fragment's answer must not depend on
        how many others its piece of the file holds."""
        from .engine import DeviceBatch
        e, t = self.engine, self.engine.torch
        if batch.n == 0:
            return t.empty(0, dtype=t.int32, device=e.device), t.empty(0, dtype=t.float32, device=e.device)
        rows = max(1, min(rows, limit // (4 * self.K)))
        cls, prob = [], []
        with e._own_stream(inputs=(batch.data, batch.off, batch.len)) as results:
            scores = t.empty((rows, self.K), dtype=t.float32, device=e.device)
            for lo in range(0, batch.n, rows):
                n = min(batch.n - lo, rows)
                e.predict(DeviceBatch(batch.data, batch.off[lo:lo + n], batch.len[lo:lo + n], n, batch.nbytes), reverse, want_scores=True, out_scores=scores)
                scores[n:].zero_()
                c, p = self.predict(scores)
                cls.append(c[:n])
                prob.append(p[:n])
            results += [t.cat(cls), t.cat(prob)]
        return tuple(results)

    def save(self, path, model=None):
        """model: the file of the linear model that the head was trained behind; load() then knows it from another."""
        with open(path, "wb") as f:
            f.write(_HDR.pack(_MAGIC, 1 if model is None else 2, self.K, self.hidden))
            if model is not None:
                f.write(model_digest(model))
            for n in _NAMES:
                self.params[n].cpu().numpy().tofile(f)

    @staticmethod
    def _header(f, path):
        """(K, hidden, the model's digest or None) from the beginning of a head file; RuntimeError for anything else."""
        raw = f.read(_HDR.size)
        if len(raw) < _HDR.size or raw[:8] != _MAGIC:
            raise RuntimeError("%s is not an opal_amd score head" % path)
        _, version, K, hidden = _HDR.unpack(raw)
        if version not in (1, 2) or not 1 <= K <= 1 << 20 or not 1 <= hidden <= 1 << 20:
            raise RuntimeError("unsupported opal_amd score head in %s" % path)
        if os.fstat(f.fileno()).st_size != _HDR.size + (version == 2) * _DIGEST + 4 * sum(int(np.prod(s)) for s in ScoreHead._shapes(K, hidden).values()):
            raise RuntimeError("truncated head file " + path)
        return K, hidden, f.read(_DIGEST) if version == 2 else None

    @staticmethod
    def _shapes(K, hidden):
        return dict(gamma=(K,), beta=(K,), w1=(hidden, K), b1=(hidden,), w2=(K, hidden), b2=(K,))

    @staticmethod
    def read(path):
        """(K, hidden, parameters) of a head file; RuntimeError for anything else."""
        with open(path, "rb") as f:
            K, hidden, _ = ScoreHead._header(f, path)
            shapes = ScoreHead._shapes(K, hidden)
            return K, hidden, {n: np.fromfile(f, dtype=np.float32, count=int(np.prod(shapes[n]))).reshape(shapes[n]) for n in _NAMES}

    @staticmethod
    def load(engine, path, model=None):
        """model: the file of the linear model that is to be used; RuntimeError when the head was trained behind another (a head that was
        saved without one is taken as it is)."""
        if model is not None:
            with open(path, "rb") as f:
                trained_behind = ScoreHead._header(f, path)[2]
            if trained_behind is not None and trained_behind != model_digest(model):
                raise RuntimeError("%s was trained behind another model than %s: train it anew (train --head) or answer without it (predict --no-head)" % (path, model))
        K, hidden, params = ScoreHead.read(path)
        return ScoreHead(engine, K, hidden, params=params)
