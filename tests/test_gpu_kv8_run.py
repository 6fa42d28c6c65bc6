"""GPU test of the 8-bit cache, the attention over it and the log probabilities together: a layer of a LLaMA by the
builtins reads documents, scores them token by token, and continues them."""
import numpy as np
import pytest

from test_gpu_kv8 import check_attention, exact_values, held_values, same
from test_gpu_logprobs import oracle

pytestmark = pytest.mark.gpu

F16 = 1
VOCAB, DIM, H, HKV, D = 517, 256, 4, 2, 64


class Layer:
    """One layer and the head, with f16 weights."""

    def __init__(self, dev, seed):
        from tensorlogic_b200.api import QTensor
        rng = np.random.default_rng(seed)

        def weight(n, k):
            return QTensor.from_blocks(dev, F16, n, k, (rng.standard_normal((n, k)) * k ** -0.5).astype(np.float16))
        self.dev = dev
        self.table = dev.tensor(rng.standard_normal((VOCAB, DIM)).astype(np.float16))
        self.norms = [dev.tensor(np.ones(DIM, np.float16)) for _ in range(2)]
        self.q, self.k, self.v = weight(H * D, DIM), weight(HKV * D, DIM), weight(HKV * D, DIM)
        self.o, self.head = weight(DIM, H * D), weight(VOCAB, DIM)

    def heads(self, ids, **where):
        from tensorlogic_b200.api import embedding, linear, rms_norm, rope
        x = embedding(self.table, ids)
        n, m = rms_norm(x, self.norms[0]), len(ids)
        q, k = (rope(linear(n, w).reshape((m, heads, D)), **where) for w, heads in ((self.q, H), (self.k, HKV)))
        return x, q, k, linear(n, self.v).reshape((m, HKV, D))

    def logits(self, x, attended, m):
        from tensorlogic_b200.api import linear, linear_residual, rms_norm
        return linear(rms_norm(linear_residual(attended.reshape((m, H * D)), self.o, x), self.norms[1]), self.head)


def check_logprobs(logits, tokens, got, top):
    for i, (lp, h, ids, best, tol) in enumerate(oracle(logits, tokens, top)):
        for g, w in [(got[0][i], lp)] + list(zip(got[3][i], best)):
            assert abs(g - w) <= tol[0] + 2.0 ** -22 * abs(w), (i, g, w)
        assert abs(got[1][i] - h) <= tol[1] and list(got[2][i]) == ids, i


def test_documents_scored_and_continued(dev):
    """Two documents are read in parts (the second with the first part dropped and read again), each scored as it is
    read; both are then continued together, greedily, across the ends of blocks.  Every stage is checked against 64 bits
    on what it was given, the cache bit for bit against all rows given to it."""
    from tensorlogic_b200.api import KVCache8, token_logprobs
    net = Layer(dev, 3)
    rng = np.random.default_rng(4)
    parts = {0: [70, 1, 51], 1: [64, 120]}
    steps, top = 72, 5
    cache = KVCache8(dev, 1, HKV, D, max_seq=300, max_batch=2)
    given = {s: [np.empty((0, HKV, D), np.float16)] * 2 for s in parts}  # the cache's rows, as they were before it
    last, scored = {}, {0: 0, 1: 0}

    def read(s, ids, at):
        """The document's next tokens (ids[0] is in hand already), and how likely each of the rest is."""
        m = len(ids) - 1
        x, q, k, v = net.heads(ids[:-1], position_offset=at)
        cache.append(0, k, v, sequence=s, position=at)
        given[s] = [np.concatenate([a[:at], t.numpy()]) for a, t in zip(given[s], (k, v))]
        out = cache.attention(0, q, H, q_pos0=at, sequence=s)
        check_attention(out.numpy(), q.numpy(), *(exact_values(a) for a in given[s]), at)
        logits = net.logits(x, out, m)
        got = token_logprobs(logits, ids[1:], top)
        check_logprobs(logits.numpy(), ids[1:], got, top)
        last[s] = int(got[2][-1][0])
        scored[s] += m

    for s, sizes in parts.items():
        at = 0
        for n in sizes:
            ids = rng.integers(0, VOCAB, n + 1)
            read(s, ids, at)
            if s == 1 and at == 0:
                read(s, ids, 0)  # once more from the start
            at += n
    assert [int(n) for n in cache.lengths[0]] == [122, 184]

    for i in range(steps):
        pos = cache.lengths[0].astype(np.int32)
        if i == 40:
            pos[0] = -1  # the first one rests for a step
        ids = [last[0], last[1]]
        x, q, k, v = net.heads(ids, positions=np.maximum(pos, 0))
        cache.append(0, k, v, positions=pos)
        out = cache.attention(0, q, H, batch=2, positions=pos)
        logits = net.logits(x, out, 2)
        greedy = logits.numpy().astype(np.float64).argmax(1)
        tokens = np.where(pos < 0, -1, greedy)
        got = token_logprobs(logits, tokens, top)
        check_logprobs(logits.numpy(), tokens, got, top)
        for s in range(2):
            if pos[s] < 0:
                assert not out.numpy()[s].any() and got[0][s] == 0
                continue
            given[s] = [np.concatenate([a, t.numpy()[s:s + 1]]) for a, t in zip(given[s], (k, v))]
            check_attention(out.numpy()[s:s + 1], q.numpy()[s:s + 1], *(exact_values(a) for a in given[s]), int(pos[s]))
            assert got[0][s] == got[3][s][0] and tokens[s] == got[2][s][0]
            last[s] = int(tokens[s])
    assert [int(n) for n in cache.lengths[0]] == [122 + steps - 1, 184 + steps]
    for s in range(2):
        for g, a in zip(cache.layer_arrays(0, s), given[s]):
            assert same(g, held_values(a))
    dev.synchronize()
