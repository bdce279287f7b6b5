"""Beam search's step against its definition in 64 bits: tokens, parents, ends and
lengths are equal, scores are sums in 64 bits rounded once. Ranks closer than
the exponentials' 32 bits tell apart do not occur in these inputs (asserted)."""
import numpy as np
import pytest

import nutllm_amd as nut
from paged_case import TYPES, decode, encode
from serving_case import beam_step, dev, space

pytestmark = pytest.mark.gpu


class Step:
    def __init__(self, gpu, scores, logits, keep, *, kind="f32", lengths=None, ended=None, eos=-1,
                 power=0.0, stride=0, offset=0):
        self.gpu = gpu
        scores = np.asarray(scores, np.float32)
        lengths, ended = (None if x is None else np.asarray(x, np.int32) for x in (lengths, ended))
        self.requests, self.beams = scores.shape
        vocab = logits.shape[-1]
        stored = encode(logits, kind)
        rows = stored.reshape(-1, vocab)
        wide = np.zeros((len(rows), stride or vocab), stored.dtype)
        wide[:, :vocab] = rows
        wide[:, vocab:] = encode(np.float32(1e4), kind)  # what stands between rows is not read
        flat = np.concatenate([wide[0, :1].repeat(offset), wide.reshape(-1)])
        self.d_logits = nut.DeviceArray(like=flat)

        class At:
            ptr, nbytes = self.d_logits.ptr.value + offset * stored.itemsize, 0
        full = lambda x, dtype: dev(np.full((self.requests, keep), x), dtype)  # noqa: E731
        self.out = [full(-9, np.int32), full(-9, np.int32), full(9.0, np.float32),
                    full(-9, np.int32), full(-9, np.int32)]
        self.d = [dev(scores, np.float32), None if lengths is None else dev(lengths),
                  None if ended is None else dev(ended)]
        old = gpu.BeamState(self.d[0], self.requests, self.beams, lengths=self.d[1],
                            ended=self.d[2])
        new = gpu.BeamState(self.out[2], self.requests, keep,
                            lengths=None if lengths is None else self.out[3],
                            ended=None if ended is None else self.out[4])
        self.work = space(gpu.beam_select_workspace(old, new, vocab))
        gpu.beam_select(old, new, At, vocab, self.out[0], self.out[1], dtype=TYPES[kind],
                        row_stride=stride, eos=eos, power=power, workspace=self.work)
        gpu.synchronize()
        self.got = [a.download(t, self.requests * keep).reshape(self.requests, keep)
                    for a, t in zip(self.out, [np.int32, np.int32, np.float32, np.int32, np.int32])]
        want, self.ranks = beam_step(scores, lengths, ended, decode(stored, kind).reshape(
            self.requests, self.beams, vocab), keep, eos, power)
        self.want = want
        self.keeps = (True, True, True, lengths is not None, ended is not None)

    def check(self):
        """Scores: float(score + logit - lse) where lse's sum has exponentials off by
        a few 2^-24 (averaged, with weights that add up to 1), and one rounding."""
        for i, (got, want) in enumerate(zip(self.got, self.want)):
            if not self.keeps[i]:
                assert np.all(got == -9)
            elif i == 2:
                live = want > -np.inf
                assert np.array_equal(got > -np.inf, live)
                assert np.all(np.abs(got[live] - want[live]) <=
                              4 * 2.0 ** -24 + 2.0 ** -24 * np.abs(want[live]))
            else:
                assert np.array_equal(got, want), (i, got, want)
        return self

    def distinct(self):
        """No two ranks that the sums' errors could turn round, or any of equal beams."""
        d = -np.diff(self.ranks, axis=1)
        assert np.all(~np.isfinite(d) | (d == 0) | (d > 1e-6)), np.nanmin(d)
        return self


def _state(rng, requests, beams, ended=0.0):
    scores = -rng.random((requests, beams)).astype(np.float32) * 5 - 3
    lengths = rng.integers(1, 50, (requests, beams)).astype(np.int32)
    return scores, lengths, (rng.random((requests, beams)) < ended).astype(np.int32)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("requests,beams,keep,vocab", [
    (1, 1, 1, 1), (1, 1, 5, 7), (3, 4, 4, 50), (2, 8, 8, 1000), (5, 2, 7, 1024), (2, 3, 3, 1031),
    (1, 4, 4, 32000), (2, 5, 64, 4099), (2, 64, 3, 300), (1, 16, 16, 65537), (1, 64, 64, 2048),
    (1, 2, 4, 262144), (1, 1, 64, 262143), (40, 1, 1, 2049),
])
@pytest.mark.parametrize("power,ended", [(0.0, 0.0), (0.7, 0.3)])
def test_step(gpu, kind, requests, beams, keep, vocab, power, ended):
    rng = np.random.default_rng(vocab + keep)
    scores, lengths, over = _state(rng, requests, beams, ended)
    logits = rng.standard_normal((requests, beams, vocab)) * 3
    Step(gpu, scores, logits, keep, kind=kind, lengths=lengths, ended=over,
         eos=min(2, vocab - 1), power=power).distinct().check()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("stride,offset", [(1000, 0), (1001, 1), (1003, 5), (1008, 7), (0, 3)])
def test_rows_that_begin_anywhere(gpu, kind, stride, offset):
    rng = np.random.default_rng(stride + offset)
    scores, lengths, _ = _state(rng, 2, 3)
    s = Step(gpu, scores, rng.standard_normal((2, 3, 997)) * 2, 6, kind=kind, stride=stride,
             offset=offset)
    s.distinct().check()


def test_without_lengths_and_ends(gpu):
    rng = np.random.default_rng(0)
    scores, _, _ = _state(rng, 3, 4)
    Step(gpu, scores, rng.standard_normal((3, 4, 100)), 4, eos=5).distinct().check()


def test_first_step(gpu):
    """One beam of each request; the others are none."""
    rng = np.random.default_rng(1)
    scores = np.full((3, 4), -np.inf, np.float32)
    scores[:, 0] = 0.0
    logits = rng.standard_normal((3, 4, 77)) * 3
    s = Step(gpu, scores, logits, 4, lengths=np.zeros((3, 4)), ended=np.zeros((3, 4)), eos=1)
    s.distinct().check()
    assert np.all(s.got[0] == np.arange(3)[:, None] * 4)


def test_fewer_candidates_than_beams(gpu):
    scores = np.array([[-1.0, -np.inf], [-np.inf, -np.inf], [np.nan, -2.0]], np.float32)
    logits = np.zeros((3, 2, 3))
    logits[:, :, 1] = 1.0
    s = Step(gpu, scores, logits, 5, lengths=np.full((3, 2), 4), ended=np.zeros((3, 2)), eos=0)
    s.check()
    assert s.got[0].tolist() == [[0, 0, 0, -1, -1], [-1] * 5, [5, 5, 5, -1, -1]]
    assert s.got[1].tolist() == [[1, 0, 2, -1, -1], [-1] * 5, [1, 0, 2, -1, -1]]
    assert s.got[4].tolist() == [[0, 1, 0, 0, 0], [0] * 5, [0, 1, 0, 0, 0]]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_masked_logits(gpu, kind):
    """Minus infinity for tokens that are not allowed: a whole part of the
    vocabulary, all but one token, all; infinite ones and NaN leave a beam none."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((1, 8, 5000)) * 2
    x[0, 0, :3000] = -np.inf
    x[0, 1] = -np.inf
    x[0, 1, 4321] = 0.5
    x[0, 2] = -np.inf
    x[0, 3, 77] = np.inf
    x[0, 4, 78] = np.nan
    x[0, 5, 100:] = -np.inf
    x[0, 6, :] = -np.inf
    x[0, 6, 9] = np.nan
    x[0, 7] -= 3e4 if kind == "f16" else 1e30
    scores = -np.arange(8, dtype=np.float32)[None] / 7 - 1
    s = Step(gpu, scores, x, 32, kind=kind)
    s.check()
    assert not set(s.got[0].ravel()) & {2, 3, 4, 6}
    only = Step(gpu, scores[:, 1:2], x[:, 1:2], 3, kind=kind).check()
    assert only.got[0].tolist() == [[0, -1, -1]] and only.got[1].tolist() == [[4321, -1, -1]]
    assert only.got[2][0, 0] == scores[0, 1]


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("vocab", [5, 64, 1025, 9000])
def test_ties_go_to_the_lowest(gpu, kind, vocab):
    """Equal logits, zeros of both signs, and beams that are the same."""
    x = np.zeros((1, 3, vocab))
    x[0, :, ::2] = -0.0
    s = Step(gpu, [[-1.0, -1.0, -1.0]], x, 4, kind=kind).check()
    assert s.got[0].tolist() == [[0, 0, 0, 0]] and s.got[1].tolist() == [[0, 1, 2, 3]]
    x[:, :, 3] = 7.0
    s = Step(gpu, [[-1.0, -1.0, -1.0]], x, 4, kind=kind).check()
    assert s.got[0].tolist() == [[0, 1, 2, 0]] and s.got[1].tolist() == [[3, 3, 3, 0]]
    rng = np.random.default_rng(3)
    y = np.broadcast_to(rng.integers(0, 4, (1, 1, vocab)).astype(float), (1, 3, vocab))
    Step(gpu, [[-1.0, -1.0, -1.0]], y, min(40, vocab), kind=kind).check()


@pytest.mark.parametrize("beams,keep,vocab", [(20, 64, 5000), (64, 64, 2048), (17, 3, 9000),
                                              (64, 9, 70000), (3, 64, 64), (33, 16, 1030)])
@pytest.mark.parametrize("levels", [1, 2, 50])
def test_many_ties(gpu, beams, keep, vocab, levels):
    """More candidates of one rank than are kept, beside ended beams and beams that are none."""
    rng = np.random.default_rng(vocab + levels)
    scores = np.full((3, beams), -2.0, np.float32)
    scores[:, 1::5] = -np.inf
    over = rng.random((3, beams)) < 0.2
    row = rng.integers(0, levels, (1, 1, vocab)).astype(float)
    Step(gpu, scores, np.broadcast_to(row, (3, beams, vocab)), keep, lengths=np.full((3, beams), 7), ended=over, eos=2,
         power=0.5).check()


@pytest.mark.parametrize("vocab", [4096, 40000])
@pytest.mark.parametrize("order", ["falling", "rising"])
def test_sorted_logits(gpu, vocab, order):
    """All of the largest in one lane's run of the vocabulary, or one wave's."""
    x = np.linspace(10, -10, vocab)[None, None]
    if order == "rising":
        x = x[..., ::-1]
    Step(gpu, [[0.0]], np.ascontiguousarray(x), 64).check()


def test_ended_beams_stay(gpu):
    """Text that has ended keeps its score and its length, and is one candidate."""
    x = np.zeros((1, 3, 10))
    x[0, 0, 4] = 30.0
    x[0, 2, 1] = 30.0
    s = Step(gpu, [[-4.0, -2.0, -3.0]], x, 3, lengths=[[5, 9, 5]], ended=[[0, 1, 0]], eos=1)
    s.check()
    assert s.got[0].tolist() == [[1, 2, 0]] and s.got[1].tolist() == [[1, 1, 4]]
    assert s.got[3].tolist() == [[9, 6, 6]] and s.got[4].tolist() == [[1, 1, 0]]
    # by score over length the long text's is the best by far, and a power below 0 turns it round
    s = Step(gpu, [[-4.0, -2.0, -3.0]], x, 3, lengths=[[5, 9, 5]], ended=[[0, 1, 0]], eos=1,
             power=1.0).check()
    assert s.got[0].tolist() == [[1, 2, 0]]
    Step(gpu, [[-4.0, -2.0, -3.0]], x, 3, lengths=[[5, 9, 5]], ended=[[0, 1, 0]], eos=1,
         power=-2.0).check()


def test_sums_of_many_logits(gpu):
    """The log-sum of 200,000 equal logits, and of one far above the others."""
    x = np.zeros((1, 2, 200000))
    x[0, 1, 150000] = 80.0
    s = Step(gpu, [[-1.0, -1.0]], x, 2).check()
    assert s.got[1].tolist() == [[150000, 0]]


@pytest.mark.parametrize("words,extra", [(1, 0), (3, 1), (4, 0), (64, 0), (1001, 3), (5000, 4)])
def test_gather(gpu, words, extra):
    """Rows by parents, twice the same one; a row without a parent stays."""
    rng = np.random.default_rng(words)
    source = rng.integers(-9, 9, (7, words + extra)).astype(np.int32)
    to = rng.integers(10, 20, (9, words + 2 * extra)).astype(np.int32)
    parents = [3, 3, 0, -1, 6, 2, 2, 2, 5]
    status, d = dev([0]), dev(to)
    gpu.beam_gather(dev(source), d, 4 * words, dev(parents), rows=9, sources=7,
                    from_stride=4 * (words + extra), to_stride=4 * (words + 2 * extra),
                    status=status)
    gpu.check_status(status)
    for i, p in enumerate(parents):
        if p >= 0:
            to[i, :words] = source[p, :words]
    assert np.array_equal(d.download(np.int32, to.size).reshape(to.shape), to)


@pytest.mark.parametrize("bad", [7, -2, 1 << 30])
def test_gather_of_rows_that_are_none(gpu, bad):
    status, d = dev([0]), dev(np.zeros((2, 8)))
    source = dev(np.arange(56).reshape(7, 8))
    gpu.beam_gather(source, d, 32, dev([bad, 1]), rows=2, sources=7, status=status)
    assert d.download(np.int32, 16).reshape(2, 8).tolist() == [[0] * 8, list(range(8, 16))]
    with pytest.raises(gpu.OutOfRange, match="parent out of range"):
        gpu.check_status(status)
    gpu.beam_gather(source, d, 32, dev([bad, 1]), rows=2, sources=7)
    gpu.synchronize()
