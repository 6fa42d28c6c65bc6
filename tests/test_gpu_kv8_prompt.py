"""GPU tests of long prompts over the 8-bit KV cache, on the tensor-memory kernel: inputs that only its arithmetic can
lose, against 64 bits."""
import numpy as np
import pytest

from test_gpu_kv8 import check_attention, exact_values

pytestmark = pytest.mark.gpu


def prompt(dev, cache, q, H, launches=2, **where):
    """Attention of a prompt's queries, and that it ran on the tensor-memory kernel (behind its image: two launches)."""
    t = dev.tensor(q)
    before = dev.launch_count
    got = cache.attention(0, t, H, **where).numpy()
    assert dev.launch_count - before == launches
    return got


@pytest.mark.parametrize("H,Hkv,D", [(32, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize("size,ahead", [(1e-3, 15), (1e-3, 17), (1e-4, 11), (1e-2, 17)])
@pytest.mark.parametrize("block", [0, 5])
def test_block_of_zeros(dev, H, Hkv, D, size, ahead, block):
    """A block whose values are all zero, with a key that outweighs each of the others 2^ahead times: the output is what
    the others add up to."""
    from tensorlogic_b200.api import KVCache8
    T = 1024
    rng = np.random.default_rng(ahead)
    k = (rng.standard_normal((T, Hkv, D)) * 0.02).astype(np.float16)
    v = ((1 + 0.1 * rng.standard_normal((T, Hkv, D))) * size).astype(np.float16)
    v[64 * block:64 * block + 64] = 0
    to = np.where(rng.random((Hkv, D)) < 0.5, 1, -1) / np.sqrt(D)
    q = (8 * np.repeat(to, H // Hkv, 0) + rng.standard_normal((T, H, D)) * 0.02).astype(np.float16)
    k[64 * block + 5] = to * (ahead * np.log(2) / 8 * np.sqrt(D))
    cache = KVCache8(dev, 1, Hkv, D, max_seq=T)
    cache.append(0, dev.tensor(k), dev.tensor(v))
    got = prompt(dev, cache, q, H)
    check_attention(got, q, exact_values(k), exact_values(v), 0)
    dev.synchronize()


def test_nothing_but_zeros(dev):
    from tensorlogic_b200.api import KVCache8
    H, Hkv, D, T = 8, 2, 128, 1000
    cache = KVCache8(dev, 1, Hkv, D, max_seq=T)
    rng = np.random.default_rng(1)
    k, q = rng.standard_normal((T, Hkv, D)), rng.standard_normal((T, H, D)).astype(np.float16)
    cache.append(0, dev.tensor(k), dev.tensor(np.zeros((T, Hkv, D))))
    assert not prompt(dev, cache, q, H).any()
    dev.synchronize()


@pytest.mark.parametrize("H,Hkv,D", [(32, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize("sign", [1, -1])
def test_largest_values(dev, H, Hkv, D, sign):
    """Values that are all the largest f16: so is their average, whatever P is rounded to."""
    from tensorlogic_b200.api import KVCache8
    T = 1000
    rng = np.random.default_rng(D)
    k = np.zeros((T, Hkv, D), np.float16)
    k[64:] = rng.standard_normal((Hkv, D)) * 0.01  # (one score in front, another behind: P of the latter rounds as one)
    v = np.full((T, Hkv, D), sign * 65504, np.float16)
    q = rng.standard_normal((T, H, D)).astype(np.float16)
    cache = KVCache8(dev, 1, Hkv, D, max_seq=T)
    cache.append(0, dev.tensor(k), dev.tensor(v))
    check_attention(prompt(dev, cache, q, H), q, exact_values(k), exact_values(v), 0)
    dev.synchronize()
