"""GPU tests of prompts over the 8-bit KV cache, against 64 bits: inputs that only the tensor-memory kernel's arithmetic can
lose, where it runs by itself, and each of its branches with either kernel asked for (option attn8_tc).

check_attention's bound holds for that kernel too.  It rounds P (half the two roundings that are allowed for: its sum is
not rounded), and P has the block's scale in it.  The key that p times its block's scale s is largest for has P >= 2^8, so
the sum is at least 2^8 / s.  A P below f16's normal range is off by 2^-25, and stands for codes up to 127: for a row of n
keys that is below n 2^-25 * 127 s / 2^8 <= n 2^-33 max|v|, at 2048 keys a fiftieth of what the other kernel's offset is
given."""
import contextlib

import numpy as np
import pytest

from test_gpu_kv8 import check_attention, exact_values, queries, rows, same

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def forced(dev, form):
    dev.set_option("attn8_tc", form)
    try:
        yield
    finally:
        dev.set_option("attn8_tc", 0)


@pytest.fixture(params=[1, 2], ids=["tcgen05", "mma"])
def form(request, dev):
    with forced(dev, request.param):
        yield request.param


def prompt(dev, cache, q, H, form=1, **where):
    """Attention of a prompt's queries, and that it ran on the tensor-memory kernel (behind its image: two launches for
    each sequence) or on the other one."""
    t = dev.tensor(q)
    before = dev.launch_count
    got = cache.attention(0, t, H, **where).numpy()
    assert dev.launch_count - before == (1 if form == 2 else 2 * where.get("batch", 1))
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


# ---- every branch on both kernels ---------------------------------------------------------------------------------

@pytest.mark.parametrize("H,Hkv,D", [(32, 4, 64), (4, 4, 128), (6, 2, 64), (20, 1, 128), (128, 1, 64)])
@pytest.mark.parametrize("I,pos0", [(2, 0), (17, 0), (64, 64), (77, 391), (130, 62), (300, 5), (3, 1000)])
def test_prompt(dev, form, H, Hkv, D, I, pos0):
    """Groups that do not fill a tile's 128 rows, and one head's worth of it; prompts shorter than a tile."""
    from tensorlogic_b200.api import KVCache8
    k, v = rows(I + pos0, pos0 + I, Hkv, D)
    q = queries(I, I, H, D)
    cache = KVCache8(dev, 1, Hkv, D, max_seq=pos0 + I + 3, max_batch=2)
    cache.append(0, dev.tensor(k), dev.tensor(v), sequence=1)
    got = prompt(dev, cache, q, H, form, q_pos0=pos0, sequence=1)
    check_attention(got, q, exact_values(k), exact_values(v), pos0)
    dev.synchronize()


@pytest.mark.parametrize("asked", [0, 1])
@pytest.mark.parametrize("I", [1, 70])
def test_groups_too_large_for_a_tile(dev, asked, I):
    from tensorlogic_b200.api import KVCache8
    H, Hkv, D = 129, 1, 64
    k, v = rows(1, I, Hkv, D)
    q = queries(1, I, H, D)
    cache = KVCache8(dev, 1, Hkv, D, max_seq=I)
    cache.append(0, dev.tensor(k), dev.tensor(v))
    with forced(dev, asked):
        got = prompt(dev, cache, q, H, 2)
    check_attention(got, q, exact_values(k), exact_values(v), 0)
    dev.synchronize()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale", [None, 0.0, -0.125, 2.0])
def test_extreme(dev, form, D, scale):
    """The largest f16 in keys, values and scale factors; blocks of keys and of values that are all zero; blocks of very
    different size side by side, sealed and open."""
    from tensorlogic_b200.api import KVCache8
    H, Hkv, T = 8, 2, 330
    k, v = rows(1, T, Hkv, D)
    k[:64] *= 2.0 ** -10
    v[:64] *= 2.0 ** -12
    v[64:128] = np.where(v[64:128] > 0, 65504, -65504)
    k[128:192], v[192:256] = 0, 0
    k[70, 0, :] = 30
    k[300, 1, :] = -30
    v[310] *= 2.0 ** -14
    q = queries(2, T, H, D)
    cache = KVCache8(dev, 1, Hkv, D, max_seq=T)
    cache.append(0, dev.tensor(k), dev.tensor(v))
    got = prompt(dev, cache, q, H, form, scale=scale)
    check_attention(got, q, exact_values(k), exact_values(v), 0, scale)
    dev.synchronize()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("I", [8, 400])
def test_scales_far_apart(dev, form, D, I):
    """In a block of large values one row of tiny ones that most of P falls on; blocks of far smaller values around it."""
    from tensorlogic_b200.api import KVCache8
    H, Hkv, T = 4, 2, 640
    k, v = (a.astype(np.float32) for a in rows(7, T, Hkv, D))
    for a in (k, v):
        a[:64] *= 30
        a[64:320] *= 1e-3
    q = queries(7, I, H, D)
    k[5] = 64 * q[0].reshape(Hkv, H // Hkv, D)[:, 0] / np.sqrt(D)
    v[5] = 1e-4
    k, v = k.astype(np.float16), v.astype(np.float16)
    cache = KVCache8(dev, 1, Hkv, D, max_seq=T)
    cache.append(0, dev.tensor(k), dev.tensor(v))
    got = prompt(dev, cache, q, H, form, q_pos0=T - I)
    check_attention(got, q, exact_values(k), exact_values(v), T - I)
    dev.synchronize()


@pytest.mark.parametrize("D", [64, 128])
def test_likely_key_of_an_open_block(dev, form, D):
    """The block that is still filling counts by 1 whatever its values are: a row of zeros in it that outweighs the rest."""
    from tensorlogic_b200.api import KVCache8
    H, Hkv, T, at, ahead = 4, 2, 360, 330, 15
    rng = np.random.default_rng(D)
    k = (rng.standard_normal((T, Hkv, D)) * 0.02).astype(np.float16)
    v = ((1 + 0.1 * rng.standard_normal((T, Hkv, D))) * 1e-3).astype(np.float16)
    to = np.where(rng.random((Hkv, D)) < 0.5, 1, -1) / np.sqrt(D)
    q = (8 * np.repeat(to, H // Hkv, 0) + rng.standard_normal((T, H, D)) * 0.02).astype(np.float16)
    k[at], v[at] = to * (ahead * np.log(2) / 8 * np.sqrt(D)), 0
    cache = KVCache8(dev, 1, Hkv, D, max_seq=T)
    cache.append(0, dev.tensor(k), dev.tensor(v))
    check_attention(prompt(dev, cache, q, H, form), q, exact_values(k), exact_values(v), 0)
    dev.synchronize()


@pytest.mark.parametrize("I,T", [(40, 60), (40, 100), (300, 300)])
def test_masked_keys(dev, form, I, T):
    """Keys and values behind a query, NaN and infinities among them, change nothing in its row; nor does what a block held
    before it was rewound."""
    from tensorlogic_b200.api import KVCache8
    H, Hkv, D = 8, 1, 64
    k, v = rows(T, T, Hkv, D)
    q = queries(T, I, H, D)
    clean, other = (KVCache8(dev, 1, Hkv, D, max_seq=T) for _ in range(2))
    clean.append(0, dev.tensor(k), dev.tensor(v))
    want = prompt(dev, clean, q, H, form, q_pos0=T - I)
    bad_k, bad_v = k.copy(), v.copy()
    bad_k[T - 1], bad_v[T - 1] = np.nan, np.inf
    other.append(0, dev.tensor(bad_k), dev.tensor(bad_v))
    got = prompt(dev, other, q, H, form, q_pos0=T - I)
    check_attention(got, q, exact_values(bad_k), exact_values(bad_v), T - I)
    assert same(got[:-1], want[:-1])
    other.append(0, dev.tensor(k), dev.tensor(v), position=0)
    assert same(prompt(dev, other, q, H, form, q_pos0=T - I), want)
    dev.synchronize()


@pytest.mark.parametrize("held", [0, 1, 64, 100, 200])
def test_cache_shorter_than_the_prompt(dev, form, held):
    """Through the C interface: queries see the keys there are, zeros where there are none, and it is reported."""
    from tensorlogic_b200 import _lib
    from tensorlogic_b200.api import KVCache8, TensorError
    H, Hkv, D, I, pos0 = 8, 2, 64, 150, 60
    k, v = rows(held + 1, held, Hkv, D)
    q = queries(held, I, H, D)
    cache = KVCache8(dev, 1, Hkv, D, max_seq=256)
    if held:
        cache.append(0, dev.tensor(k), dev.tensor(v))
    mark = np.full((I + 1, H, D), 7, np.float16)
    tq, out = dev.tensor(q), dev.tensor(mark)
    dev.synchronize()
    _lib.check(dev.lib.tlc_attention8(dev.handle, cache.handle, 0, tq.ptr, out.ptr, 1, I, H, 0, pos0, None, 0, 0.125))
    with pytest.raises(TensorError) as e:
        dev.synchronize()
    assert e.value.code == _lib.ERR_INDEX
    got = out.numpy()
    assert same(got[I], mark[I])
    if held:
        check_attention(got[:I], q, exact_values(k), exact_values(v), pos0, 0.125)
    else:
        assert not got[:I].any()
    dev.synchronize()


def test_two_sequences_in_place(dev, form):
    """A batch, a sequence after the other through one image; the output over the queries."""
    from tensorlogic_b200 import _lib
    from tensorlogic_b200.api import KVCache8
    H, Hkv, D, I, pos0 = 6, 2, 128, 90, 40
    data = [rows(b, pos0 + I, Hkv, D) for b in range(2)]
    cache = KVCache8(dev, 2, Hkv, D, max_seq=140, max_batch=3)
    for b, (k, v) in enumerate(data):
        cache.append(1, dev.tensor(k), dev.tensor(v), sequence=b + 1)
    q = queries(3, 2 * I, H, D)
    t = dev.tensor(q)
    _lib.check(dev.lib.tlc_attention8(dev.handle, cache.handle, 1, t.ptr, t.ptr, 2, I, H, 1, pos0, None, 0, D ** -0.5))
    got = t.numpy()
    for b, (k, v) in enumerate(data):
        check_attention(got[b * I:(b + 1) * I], q[b * I:(b + 1) * I], exact_values(k), exact_values(v), pos0)
    dev.synchronize()


def test_which_kernel_runs(dev):
    """By cost: a long prompt on the tensor-memory kernel, for rows of either size, a short one on the other."""
    from tensorlogic_b200 import _lib
    from tensorlogic_b200.api import KVCache8, TensorError
    for H, Hkv, D, I, form in ((32, 4, 64, 1024, 1), (8, 2, 128, 1024, 1), (32, 4, 64, 20, 2), (8, 2, 128, 20, 2)):
        cache = KVCache8(dev, 1, Hkv, D, max_seq=I)
        k, v = rows(I, I, Hkv, D)
        cache.append(0, dev.tensor(k), dev.tensor(v))
        prompt(dev, cache, queries(I, I, H, D), H, form)
    for wrong in (-1, 3):
        with pytest.raises(TensorError) as e:
            dev.set_option("attn8_tc", wrong)
        assert e.value.code == _lib.ERR_INVALID_OPERATION
    dev.synchronize()


@pytest.mark.parametrize("H,Hkv,D", [(32, 4, 64), (8, 2, 128)])
def test_first_prompt_in_a_capture(dev, H, Hkv, D):
    """A cache's first long prompt, in a graph: it runs on the kernel that it runs on outside of one, and allocates nothing."""
    import torch
    from tensorlogic_b200 import _lib
    from tensorlogic_b200.api import KVCache8
    I = 900
    k, v = rows(2, I, Hkv, D)
    q = queries(2, I, H, D)
    cache = KVCache8(dev, 1, Hkv, D, max_seq=1000, max_batch=2)
    cache.append(0, dev.tensor(k), dev.tensor(v), sequence=1)
    tq, out = torch.tensor(q, device="cuda"), torch.zeros(I, H, D, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    dev.synchronize()
    before = dev.launch_count
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(dev.stream)):
        _lib.check(dev.lib.tlc_attention8(dev.handle, cache.handle, 0, tq.data_ptr(), out.data_ptr(), 1, I, H, 1, 0, None, 0, D ** -0.5))
    assert dev.launch_count - before == 2
    g.replay()
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    check_attention(got, q, exact_values(k), exact_values(v), 0)
    out.zero_()
    torch.cuda.synchronize()
    free = dev.mem_info()[0]
    _lib.check(dev.lib.tlc_attention8(dev.handle, cache.handle, 0, tq.data_ptr(), out.data_ptr(), 1, I, H, 1, 0, None, 0, D ** -0.5))
    dev.synchronize()
    assert dev.mem_info()[0] == free
    assert same(out.cpu().numpy(), got)


def test_bytes_of_a_small_cache(dev):
    """What a cache of 64 rows allocates is its workspace: one part for each cluster that leaves a part, below 2 MB."""
    from tensorlogic_b200.api import KVCache8
    dev.synchronize()
    free = dev.mem_info()[0]
    held = [KVCache8(dev, 1, 1, 128, max_seq=64) for _ in range(16)]
    dev.synchronize()
    assert free - dev.mem_info()[0] <= 16 * 2**21
    del held


@pytest.mark.parametrize("H,Hkv,D", [(32, 32, 128), (32, 4, 64), (160, 1, 64)])
def test_many_items_are_not_cut_finer(dev, H, Hkv, D):
    """Twice the prompt is four times the work.  Where warps are filled many times over, an item stays with few of them: its
    results are merged each time, not once."""
    import torch
    from tensorlogic_b200.api import KVCache8
    T = 2048
    cache = KVCache8(dev, 1, Hkv, D, max_seq=T)
    k, v = rows(1, T, Hkv, D)
    cache.append(0, dev.tensor(k), dev.tensor(v))
    stream = torch.cuda.ExternalStream(dev.stream)

    def took(I):
        q = dev.tensor(queries(1, I, H, D))
        times = []
        for _ in range(6):
            with torch.cuda.stream(stream):
                start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                start.record()
                cache.attention(0, q, H)
                end.record()
            dev.synchronize()
            times.append(start.elapsed_time(end))
        return min(times)

    with forced(dev, 2):  # (the third group is too large for the other kernel anyway)
        assert took(T) <= 8 * took(T // 2)
    dev.synchronize()


@pytest.mark.parametrize("H,Hkv,D", [(32, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize("I,T", [(1, 700), (1, 20000), (60, 700)])
def test_largest_values_of_a_token(dev, H, Hkv, D, I, T):
    """The same on the other kernel: one warp, warps, CTAs and clusters that share the keys."""
    from tensorlogic_b200.api import KVCache8
    rng = np.random.default_rng(D)
    k = (rng.standard_normal((T, Hkv, D)) * 0.01).astype(np.float16)
    q = queries(I, I, H, D)
    for value in (65504, -65504):
        v = np.full((T, Hkv, D), value, np.float16)
        cache = KVCache8(dev, 1, Hkv, D, max_seq=T)
        cache.append(0, dev.tensor(k), dev.tensor(v))
        check_attention(prompt(dev, cache, q, H, 2, q_pos0=T - I), q, exact_values(k), exact_values(v), T - I)
    dev.synchronize()
