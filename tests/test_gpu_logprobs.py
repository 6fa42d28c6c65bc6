"""GPU tests of the log probabilities of tokens against 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def oracle(x, targets, top):
    """Per row, in 64 bits: log probability, entropy, the likeliest ids and theirs, and how far f32 may be off.

    A thread adds 64 exponentials, each good to 2^-21 (ex2 and the rounding of its argument), in four chains, and
    5 + 16 partial sums follow: S is off by less than 2^-21 + 40 * 2^-24 < 2^-18 of itself, and so is sum e t of
    sum e |t|.  ln S takes that over as it is, H once with each, and each result is rounded a few times."""
    out = []
    for row, t in zip(x.astype(np.float64), targets):
        at = np.flatnonzero(np.isfinite(row))
        if not at.size:
            lp, h, ids, best, tol = -np.inf, 0.0, [], [], (0.0, 0.0)
        else:
            v = row[at]
            m = v.max()
            e = np.exp(v - m)
            lse = m + np.log(e.sum())
            p = e / e.sum()
            h = float(np.log(e.sum()) - (p * (v - m)).sum())
            order = np.lexsort((at, -v))[:top]
            ids, best = list(at[order]), list(v[order] - lse)
            lp = row[t] - lse if 0 <= t < row.size and np.isfinite(row[t]) else -np.inf
            tol = (2.0 ** -18, 2.0 ** -18 * (2 + 2 * (p * (m - v)).sum()) + 2.0 ** -21 * h)
        if t == -1:
            lp = 0.0
        ids += [-1] * (top - len(ids))
        best += [-np.inf] * (top - len(best))
        out.append((lp, h, ids, best, tol))
    return out


def check(dev, x, targets, top):
    from tensorlogic_b200.api import token_logprobs
    got = token_logprobs(dev.tensor(x), targets, top)
    assert got[2].shape == got[3].shape == (x.shape[0], top)
    for i, (lp, h, ids, best, tol) in enumerate(oracle(x, targets, top)):
        for g, w in [(got[0][i], lp)] + list(zip(got[3][i], best)):
            assert g == w if not np.isfinite(w) else abs(g - w) <= tol[0] + 2.0 ** -22 * abs(w), (i, g, w)
        assert abs(got[1][i] - h) <= tol[1], (i, got[1][i], h)
        assert list(got[2][i]) == ids, i
    return got


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 2), (3, 7), (2, 8), (5, 333), (1, 32000), (2, 32001), (70, 4097),
                                        (3, 100003), (1, 262144), (2, 300001), (160, 32768), (300, 513)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_rows(dev, rows, vocab, top):
    rng = np.random.default_rng(rows * vocab + top)
    x = (rng.standard_normal((rows, vocab)) * rng.uniform(0.5, 6, (rows, 1))).astype(np.float16)
    targets = rng.integers(0, vocab, rows)
    targets[::2] = x[::2].argmax(1)
    check(dev, x, targets, top)
    dev.synchronize()


@pytest.mark.parametrize("vocab", [31, 1000, 32003, 70001])
def test_odd_rows(dev, vocab):
    """Masks that leave much, little or nothing; the lowest f16 as a mask; ties; NaN; a row that is certain."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((16, vocab)).astype(np.float16)
    x[0] = -np.inf                                   # nothing left
    x[1] = np.nan
    x[2, 1:] = -np.inf                               # one
    x[3, rng.random(vocab) < 0.95] = -np.inf
    x[4] = -65504                                    # all the lowest value: even
    x[5, ::2] = -65504
    x[6] = 0                                         # all equal: ids in order
    x[7] = np.where(np.arange(vocab) % 2, 0.0, -0.0)  # equal too
    x[8] = rng.integers(0, 3, vocab)                 # ties everywhere
    x[9, 5], x[9, 7], x[9, 9] = np.nan, np.inf, -np.inf
    x[10] = np.arange(vocab)[::-1] * (60000.0 / vocab)  # sorted
    x[11] = np.arange(vocab) * (60000.0 / vocab)
    x[12, 17] = 65504                                # certain
    x[13] = 60000 + rng.standard_normal(vocab) * 50  # large
    x[14, 20:] = -np.inf                             # fewer than 32
    targets = rng.integers(0, vocab, 16)
    targets[2], targets[3], targets[12], targets[15], targets[9] = 0, x[3].argmax(), 17, -1, 7
    check(dev, x, targets, 32 if vocab >= 32 else 20)
    check(dev, x, targets, 3)
    dev.synchronize()


def test_parts_on_their_own(dev):
    """Every output may be left out; rows behind the last one stay as they were; a target outside is reported."""
    import torch
    from tensorlogic_b200 import _lib
    from tensorlogic_b200.api import TensorError, token_logprobs
    rows, vocab, top = 4, 1001, 3
    x = torch.randn(rows, vocab, device="cuda").half()
    targets = torch.tensor([5, -1, 1000, 0], dtype=torch.int32, device="cuda")
    want = token_logprobs(dev.tensor(x.cpu().numpy()), targets.cpu().numpy(), top)
    torch.cuda.synchronize()

    def call(lp, h, ids, best, k=top, t=targets):
        p = [a.data_ptr() if a is not None else None for a in (lp, h, ids, best)]
        return dev.lib.tlc_token_logprobs(dev.handle, x.data_ptr(), rows, vocab, t.data_ptr() if t is not None else None, k, *p)

    def fresh():
        out = [torch.full((rows + 1,), 7.0, device="cuda"), torch.full((rows + 1,), 7.0, device="cuda"),
               torch.full((rows + 1, top), 7, dtype=torch.int32, device="cuda"), torch.full((rows + 1, top), 7.0, device="cuda")]
        torch.cuda.synchronize()
        return out
    for keep in ((1, 1, 1, 1), (1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 1), (0, 1, 1, 1)):
        out = fresh()
        a = [o if k else None for o, k in zip(out, keep)]
        assert call(*a, k=top if keep[2] else 0, t=targets if keep[0] else None) == 0
        dev.synchronize()
        for o, k, w in zip(out, keep, want):
            # (without alternatives the sums are added in another order: each is off by 2^-18 at most, see oracle())
            assert np.allclose(o[:rows].cpu().numpy(), w, rtol=2.0 ** -16, atol=2.0 ** -17) if k else (o == 7).all()
            assert (o[rows] == 7).all()
    out = fresh()
    assert call(None, None, None, None, k=0, t=None) == 0
    bad = torch.tensor([5, -2, 1001, 2**31 - 1], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    assert call(*out, t=bad) == 0
    with pytest.raises(TensorError) as e:
        dev.synchronize()
    assert e.value.code == _lib.ERR_INDEX and "target" in str(e.value)
    lp = out[0].cpu().numpy()
    assert lp[0] == want[0][0] and np.isnan(lp[1:4]).all() and lp[4] == 7
    assert np.array_equal(out[1][:rows].cpu().numpy(), want[1])
    dev.synchronize()


@pytest.mark.parametrize("offset", [1, 3, 7])
def test_unaligned_logits(dev, offset):
    """A view that starts anywhere in an array, and ends with it."""
    import torch
    from tensorlogic_b200 import _lib
    from tensorlogic_b200.api import token_logprobs
    rows, vocab = 3, 2045
    whole = torch.randn(offset + rows * vocab, device="cuda").half()
    x = whole[offset:]
    ids, best = torch.empty(rows, 4, dtype=torch.int32, device="cuda"), torch.empty(rows, 4, device="cuda")
    h = torch.empty(rows, device="cuda")
    torch.cuda.synchronize()
    _lib.check(dev.lib.tlc_token_logprobs(dev.handle, x.data_ptr(), rows, vocab, None, 4, None, h.data_ptr(), ids.data_ptr(), best.data_ptr()))
    dev.synchronize()
    want = token_logprobs(dev.tensor(x.cpu().numpy().reshape(rows, vocab)), None, 4)
    # (sums are added in another order)
    assert np.array_equal(ids.cpu().numpy(), want[2]) and np.allclose(best.cpu().numpy(), want[3], rtol=0, atol=2.0 ** -17)
    assert want[0] is None and np.allclose(h.cpu().numpy(), want[1], rtol=2.0 ** -16)


def test_refusals(dev):
    from tensorlogic_b200 import _lib
    from tensorlogic_b200.api import TensorError, token_logprobs
    x = dev.tensor(np.zeros((2, 10), np.float16))
    out = dev.empty((256,))
    f = dev.lib.tlc_token_logprobs

    def call(logits=x.ptr, rows=2, vocab=10, targets=None, k=0, lp=None, h=out.ptr, ids=None, best=None):
        return f(dev.handle, logits, rows, vocab, targets, k, lp, h, ids, best)
    bad, dim = _lib.ERR_INVALID_OPERATION, _lib.ERR_INVALID_DIMENSION
    assert call(logits=None) == bad and call(lp=out.ptr) == bad and call(k=33, ids=out.ptr, best=out.ptr) == bad
    assert call(k=-1) == bad and call(k=2) == bad and call(k=2, ids=out.ptr) == bad and call(logits=x.ptr + 1) == bad
    assert call(rows=-1) == dim and call(vocab=0) == dim and call(rows=2**31 - 1) == dim and call(vocab=2**31 - 1) == dim
    assert call(rows=0) == 0 and call() == 0
    for tokens in ([0], [0, 10], [-2, 0]):
        with pytest.raises(TensorError):
            token_logprobs(x, tokens)
    with pytest.raises(TensorError):
        token_logprobs(x, [0, 1], top_k=33)
    dev.synchronize()


@pytest.mark.parametrize("vocab", [131600, 8 * 16384 + 8 * 8 * 31, 140001])
def test_short_last_slice(dev, vocab):
    """Slices that end with a few pieces: the best logits before them, in them, and everywhere."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((4, vocab)).astype(np.float16)
    x[1] = np.arange(vocab) * (50.0 / vocab)
    x[2] = np.arange(vocab)[::-1] * (50.0 / vocab)
    x[3] = 1
    for top in (1, 32):
        check(dev, x, rng.integers(0, vocab, 4), top)
    dev.synchronize()


@pytest.mark.parametrize("top", [0, 5])
def test_far_into_memory(dev, top):
    """The last rows of more than 2^31 logits."""
    import torch
    from tensorlogic_b200 import _lib
    rows, vocab, last = 68000, 32000, 3
    x = torch.zeros(rows, vocab, dtype=torch.float16, device="cuda")
    x[-last:] = torch.randn(last, vocab, device="cuda").half() * 3
    t = torch.arange(rows, dtype=torch.int32, device="cuda") % vocab
    lp, h, best = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"), torch.empty(rows, 5, device="cuda")
    ids = torch.empty(rows, 5, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    _lib.check(dev.lib.tlc_token_logprobs(dev.handle, x.data_ptr(), rows, vocab, t.data_ptr(), top, lp.data_ptr(), h.data_ptr(),
                                          ids.data_ptr() if top else None, best.data_ptr() if top else None))
    dev.synchronize()
    host = [a[-last:].cpu().numpy() for a in (x, t, lp, h, ids, best)]
    for i, (p, e, at, b, tol) in enumerate(oracle(host[0], host[1], top)):
        assert abs(host[2][i] - p) <= tol[0] + 2.0 ** -22 * abs(p) and abs(host[3][i] - e) <= tol[1]
        if top:
            assert list(host[4][i]) == at and all(abs(g - w) <= tol[0] + 2.0 ** -22 * abs(w) for g, w in zip(host[5][i], b))
    even = np.log(vocab)
    assert abs(float(lp[0]) + even) <= 2.0 ** -18 + 2.0 ** -22 * even and (lp[:-last] == lp[0]).all() and (h[:-last] == h[0]).all()


@pytest.mark.parametrize("rows,vocab", [(36, 100003), (18, 151937), (48, 151936), (24, 64001), (60, 64000), (20, 32003), (100, 100000)])
@pytest.mark.parametrize("top", [0, 20])
def test_many_rows(dev, rows, vocab, top):
    """Rows shared out over every number of CTAs, and more of them than there is room for at once."""
    rng = np.random.default_rng(rows + vocab)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float16)
    x[rng.random((rows, vocab)) < 0.2] = -np.inf
    x[::5, vocab // 3:] = -np.inf                     # slices with nothing in them
    check(dev, x, rng.integers(0, vocab, rows), top)
    dev.synchronize()
