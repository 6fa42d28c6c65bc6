"""What the 8-bit KV cache and the token log probabilities refuse before anything reaches a GPU."""
import types

import numpy as np
import pytest

from tensorlogic_b200 import _lib
from tensorlogic_b200.api import KVCache8, Tensor, token_logprobs


class _Lib:
    """Every call succeeds and is written down."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def fake():
    return types.SimpleNamespace(lib=_Lib(), handle=1, _slot=(1, 4096), _slot_at=0, synchronize=lambda: None)


def _tensor(dev, shape):
    t = Tensor.__new__(Tensor)
    t.dev, t.shape, t.size, t.ptr, t._buf = dev, tuple(shape), int(np.prod(shape)), 4096, None
    return t


def test_null_context_is_refused(lib):
    for name in ("tlc_kvcache8_create", "tlc_kvcache8_append", "tlc_kvcache8_rows", "tlc_attention8", "tlc_token_logprobs"):
        args = [t() if t in (_lib.i32, _lib.f32) else None for t in _lib.PROTOTYPES[name][1]]
        assert getattr(lib, name)(*args) == _lib.ERR_INVALID_OPERATION and b"null context" in lib.tlc_last_error(), name
    assert lib.tlc_kvcache8_destroy(None) == 0


def test_cache_refusals(fake):
    cache = KVCache8(fake, 2, 2, 64, max_seq=100, max_batch=3)
    one = lambda n: _tensor(fake, (n, 2, 64))  # noqa: E731
    cache.append(0, one(40), one(40), sequence=1)
    assert list(cache.lengths[0]) == [0, 40, 0] and not cache.lengths[1].any()
    made = len(fake.lib.calls)

    def refused(code, f, *a, **k):
        with pytest.raises(_lib.TensorError) as e:
            f(*a, **k)
        assert e.value.code == code

    shape, index = _lib.ERR_SHAPE_MISMATCH, _lib.ERR_INDEX
    refused(shape, cache.append, 0, _tensor(fake, (100,)), _tensor(fake, (100,)))
    refused(shape, cache.append, 0, one(1), one(2))
    refused(index, cache.append, 2, one(1), one(1))
    refused(index, cache.append, -1, one(1), one(1))
    refused(shape, cache.append, 0, one(1), one(1), sequence=3)
    refused(shape, cache.append, 0, one(3), one(3), sequence=1, positions=[0, 0, 0])
    refused(index, cache.append, 0, one(1), one(1), position=1)                # a gap
    refused(index, cache.append, 0, one(1), one(1), position=-1)
    refused(shape, cache.append, 0, one(3), one(3), positions=[0, 40])
    refused(index, cache.append, 0, one(3), one(3), positions=[0, 41, -1])     # a gap in one of them
    refused(shape, cache.attention, 0, one(1), 3)
    refused(shape, cache.attention, 0, one(1), 2, batch=0)
    refused(shape, cache.attention, 0, one(3), 2, batch=3, sequence=1)
    refused(index, cache.attention, 0, one(1), 2)                              # nothing there
    refused(index, cache.attention, 0, one(2), 2, q_pos0=39, sequence=1)
    refused(index, cache.attention, 0, one(3), 2, batch=3, positions=[-1, 40, -1])
    refused(shape, cache.attention, 0, one(3), 2, batch=3, positions=[-1, 39])
    refused(index, cache.layer_arrays, 5)
    refused(shape, cache.layer_arrays, 0, 3)
    assert len(fake.lib.calls) == made  # nothing was called
    assert list(cache.lengths[0]) == [0, 40, 0]
    cache.append(0, one(3), one(3), positions=[0, 20, -1])
    assert list(cache.lengths[0]) == [1, 21, 0]
    cache.append(0, one(5), one(5), sequence=1, position=7)
    assert list(cache.lengths[0]) == [1, 12, 0]


def test_logprob_refusals(fake):
    x = _tensor(fake, (2, 10))
    for tokens, top in (([0], 0), ([0, 10], 0), ([-2, 0], 0), ([0, 1], 33), ([0, 1], -1)):
        with pytest.raises(_lib.TensorError):
            token_logprobs(x, tokens, top)
    assert not any(name == "tlc_token_logprobs" for name, _ in fake.lib.calls)


def test_shapes_of_nothing(fake):
    """No rows is no error; no vocabulary, or a length that no sequence can have, is one."""
    lp, entropy, ids, best = token_logprobs(_tensor(fake, (0, 10)), [], 3)
    assert lp.shape == entropy.shape == (0,) and ids.shape == best.shape == (0, 3)
    with pytest.raises(_lib.TensorError):
        token_logprobs(_tensor(fake, (2, 0)), [0, 0])
    cache = KVCache8(fake, 1, 2, 64, max_seq=100)
    for n in (-1, 101):
        with pytest.raises(_lib.TensorError) as e:
            cache.layer_arrays(0, 0, n)
        assert e.value.code == _lib.ERR_INDEX


def test_tensors_of_another_context_are_refused(fake):
    other = types.SimpleNamespace(**vars(fake))
    cache = KVCache8(fake, 1, 2, 64, max_seq=100)
    mine, theirs = _tensor(fake, (1, 2, 64)), _tensor(other, (1, 2, 64))
    cache.append(0, mine, mine)
    for call in (lambda: cache.append(0, mine, theirs), lambda: cache.append(0, theirs, mine), lambda: cache.attention(0, theirs, 2)):
        with pytest.raises(_lib.TensorError) as e:
            call()
        assert e.value.code == _lib.ERR_DEVICE
    assert list(cache.lengths[0]) == [1]


@pytest.mark.parametrize("wrong", [2**32, 2**32 + 5, 2**63 - 1, -2**32 + 5, 2**64, 5.5, np.nan, np.uint64(2**63 + 5), np.float32(2**33)])
def test_indices_are_checked_before_they_are_cut(fake, wrong):
    """A position or a token that 32 bits do not hold is out of bounds (or, negative, no position), not what is left of it."""
    cache = KVCache8(fake, 1, 2, 64, max_seq=100, max_batch=2)
    one = lambda n: _tensor(fake, (n, 2, 64))  # noqa: E731
    cache.append(0, one(40), one(40), sequence=0)
    cache.append(0, one(40), one(40), sequence=1)
    made = len(fake.lib.calls)
    none = wrong == -2**32 + 5  # any negative position: no row
    for both in (np.array([40, wrong]), [40, wrong]):
        for call in (lambda: cache.append(0, one(2), one(2), positions=both),
                     lambda: cache.attention(0, one(2), 2, batch=2, positions=np.asarray(both) - 1)):
            if not none:
                with pytest.raises(_lib.TensorError) as e:
                    call()
                assert e.value.code == _lib.ERR_INDEX
    with pytest.raises(_lib.TensorError) as e:
        token_logprobs(_tensor(fake, (2, 10)), [3, wrong])
    assert e.value.code == _lib.ERR_INDEX
    assert len(fake.lib.calls) == made and list(cache.lengths[0]) == [40, 40]
    if none:
        cache.append(0, one(2), one(2), positions=np.array([40, wrong]))
        assert list(cache.lengths[0]) == [41, 40]


def test_negative_positions_stay_negative(fake, monkeypatch):
    """What reaches the GPU for a position far below zero is below zero too."""
    from tensorlogic_b200 import api
    sent = []
    monkeypatch.setattr(api, "_upload_i32", lambda dev, a: sent.append(a) or types.SimpleNamespace(ptr=4096))
    cache = KVCache8(fake, 1, 2, 64, max_seq=100, max_batch=3)
    three = _tensor(fake, (3, 2, 64))
    cache.append(0, three, three, positions=np.array([0, -2**32 + 5, -1]))
    cache.attention(0, three, 2, batch=3, positions=np.array([0, -2**32 + 5, -2**63]))
    cache.append(0, three, three, positions=np.array([1.0, -1.0, -1.0]))  # whole numbers, whatever holds them
    assert [a.dtype for a in sent] == [np.int32] * 3
    assert [list(a) for a in sent] == [[0, -1, -1], [0, -1, -1], [1, -1, -1]]
    assert list(cache.lengths[0]) == [2, 0, 0]


def test_tokens_of_any_integer_type(fake, monkeypatch):
    from tensorlogic_b200 import api
    sent = []
    monkeypatch.setattr(api, "_upload_i32", lambda dev, a: sent.append(a) or types.SimpleNamespace(ptr=4096))
    for t in (np.int8, np.uint8, np.int64, np.uint64):
        token_logprobs(_tensor(fake, (2, 10)), np.array([3, 9], t))
    assert all(a.dtype == np.int32 and list(a) == [3, 9] for a in sent) and len(sent) == 4


@pytest.mark.parametrize("wrong", [-1, -2**32, -2**32 + 3, 2**32, 2.5])
def test_a_single_position_is_checked_whole_too(fake, wrong):
    cache = KVCache8(fake, 1, 2, 64, max_seq=100)
    rows = _tensor(fake, (5, 2, 64))
    cache.append(0, rows, rows)
    made = len(fake.lib.calls)
    for call in (lambda: cache.append(0, rows, rows, position=wrong), lambda: cache.attention(0, _tensor(fake, (2, 2, 64)), 2, q_pos0=wrong)):
        with pytest.raises(_lib.TensorError) as e:
            call()
        assert e.value.code == _lib.ERR_INDEX
    assert len(fake.lib.calls) == made and list(cache.lengths[0]) == [5]
    cache.append(0, rows, rows, position=np.int64(5))
    assert list(cache.lengths[0]) == [10]
