"""What the 8-bit scores cost the selection, against the same bound without roundings (CPU: the kernels' selections equal the
oracle's)."""
import numpy as np
import pytest

from oracle import sparse as S


def _case(seed, pages, page, group, d, spread, size):
    """Queries of a row's heads and keys of pages whose channels differ in size; some keys lean towards the queries."""
    rng = np.random.default_rng(seed)
    wide = np.exp(spread * rng.standard_normal(d))
    wide /= np.sqrt((wide ** 2).mean())
    q = size * rng.standard_normal((group, d))
    keys = rng.standard_normal((pages, page, d)) * wide
    lean = rng.random((pages, page, 1)) < 0.01
    keys = np.where(lean, keys + 0.3 * q.mean(0) * wide, keys)
    return q, keys


def _bounds(q, keys):
    """The unrounded bound of each page, its highest over the heads; how far each page's 8-bit score may be from it; scores."""
    hi, lo = keys.max(1), keys.min(1)
    bound = np.maximum(q[:, None] * hi, q[:, None] * lo).sum(-1)
    got = [S.summary(k[None]) for k in keys]
    codes, scales = np.stack([c[0] for c, _ in got]), np.array([s[0] for _, s in got])
    _, unit = S.codes(q)
    # a code is within half a unit of its value (the largest, up to 127.99 units, within one unit of its own 127): a query's
    # rounding moves every channel's product by that times the larger bound, a bound's by that times the rounded query
    # (|q| + half a unit); the score's two products are rounded in f32
    off_q = np.where(np.abs(q) > 127 * unit[:, None], 1.0, 0.5) * unit[:, None]
    edge = np.maximum(np.abs(hi), np.abs(lo))
    off_k = np.where(edge > 127 * scales[:, None], 1.0, 0.5) * scales[:, None]
    far = (off_q[:, None] * edge + (np.abs(q) + off_q)[:, None] * off_k).sum(-1)
    far += 2.0 ** -22 * (np.abs(q)[:, None] * edge).sum(-1)
    return bound.max(0), far.max(0), S.scores(q, codes, scales).astype(np.float64)


CASES = [(pages, page, group, d, spread, size) for pages, page in ((200, 16), (600, 16), (80, 64))
         for group, d in ((8, 128), (1, 64)) for spread, size in ((0.5, 2.0), (1.0, 1.0))]


@pytest.mark.parametrize("pages,page,group,d,spread,size", CASES)
def test_pages_that_stand_out_are_kept(pages, page, group, d, spread, size):
    """A page whose unrounded bound is above another's by more than both scores may be off is never left for it."""
    for seed in range(4):
        q, keys = _case(seed, pages, page, group, d, spread, size)
        bound, far, score = _bounds(q, keys)
        assert (np.abs(score - bound) <= far).all()
        budget = pages // 8
        kept = S.select(score.astype(np.float32), pages, budget + 1, 0, 1)[:-1]  # (the last one is the row's own)
        left = np.setdiff1d(np.arange(pages - 1), kept)
        assert len(kept) == budget
        assert (bound[left] - far[left]).max() <= (bound[kept] + far[kept]).min()


@pytest.mark.parametrize("pages,page,group,d,spread,size", CASES)
def test_the_kept_bounds_add_up_to_nearly_the_best(pages, page, group, d, spread, size):
    """Of the unrounded bounds' sum over the pages that the unrounded bound keeps, the 8-bit selection loses at most what the
    scores of the pages that differ are off."""
    for seed in range(4):
        q, keys = _case(seed, pages, page, group, d, spread, size)
        bound, far, score = _bounds(q, keys)
        budget = pages // 8
        best = S.select(bound, pages, budget + 1, 0, 1)[:-1]
        kept = S.select(score.astype(np.float32), pages, budget + 1, 0, 1)[:-1]
        lost, won = np.setdiff1d(best, kept), np.setdiff1d(kept, best)
        assert len(lost) == len(won)
        assert bound[best].sum() - bound[kept].sum() <= far[lost].sum() + far[won].sum()
