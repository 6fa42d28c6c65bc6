"""GPU tests of the 8-bit KV cache: what it holds, bit for bit, and the attention over it against 64 bits."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

BLOCK = 64


# ---- the definition, in numpy ---------------------------------------------------------------------------------

def finite(x):
    x = x.astype(np.float16).copy()
    x[np.isnan(x)] = 0
    x[np.isposinf(x)] = 65504
    x[np.isneginf(x)] = -65504
    return x


def held_values(rows):
    """f16 [T, heads, D] as the cache holds them: full blocks as q * (a / 127) in f32, rounded to f16.  127 x / a of two
    f16 lies on a border or 2^-20 of its power of two away from it, which 64 bits tell apart."""
    x = finite(rows)
    for b in range(x.shape[0] // BLOCK):
        s = slice(b * BLOCK, (b + 1) * BLOCK)
        a = np.abs(x[s].astype(np.float64)).max(axis=(0, 2), keepdims=True)
        q = np.rint(127 * x[s].astype(np.float64) / np.where(a > 0, a, 1)).astype(np.int32)  # (a code has no -0)
        x[s] = (q.astype(np.float32) * (a.astype(np.float32) / np.float32(127))).astype(np.float16)
    return x


def exact_values(rows):
    """The same in 64 bits, not rounded to f16: what the attention's products see."""
    x = finite(rows).astype(np.float64)
    for b in range(x.shape[0] // BLOCK):
        s = slice(b * BLOCK, (b + 1) * BLOCK)
        a = np.abs(x[s]).max(axis=(0, 2), keepdims=True)
        x[s] = np.where(a > 0, np.rint(127 * x[s] / np.where(a > 0, a, 1)) * a / 127, 0)
    return x


def check_attention(got, q, k, v, pos0, scale=None):
    """out[i] of queries at pos0 + i over keys 0 .. pos0 + i, element by element.

    What the kernel rounds: P to f16 (2^-11 of each p, in numerator and sum alike: 2 * 2^-11 of sum p |v| / sum p), the
    output to f16 (2^-11 of itself, or half the smallest subnormal).  In f32: a score is a sum of D products of q with
    codes + 128 (at most 255) in steps of 16, each step good to 2^-23 of what has been added up -- below
    (D / 16 + 4) 2^-23 * 255 / 127 * sum |q| max|k| scale -- and e^x itself to 2^-21; both act on p.  The second product
    adds p (code + 128), all of one sign, to be taken off as 128 sum p: in a step of 16 the products are aligned to the
    largest and cut, so that each of a block's 64 may lose 2^-23 of at most 255 sum p, and so may each of eleven additions
    of sum p and the four that join them.  A code is worth max|v| / 127 -- below 80 * 2^-23 * 255 / 127 * max|v| whatever the
    values that count (they may all be zero)."""
    I, H, D = q.shape
    G = H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    worst = 0.0
    for h in range(H):
        kh, vh, qh = k[:, h // G], v[:, h // G], q[:, h].astype(np.float64)
        s = scale * (qh @ kh.T)
        s[np.arange(kh.shape[0])[None, :] > pos0 + np.arange(I)[:, None]] = -np.inf
        p = np.exp(s - s.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        want, size = p @ vh, p @ np.abs(vh)
        score = (D / 16 + 4) * 2.0 ** -23 * 255 / 127 * abs(scale) * np.abs(qh).sum(1, keepdims=True) * np.abs(kh).max() + 2.0 ** -21
        tol = 2.0 ** -11 * np.abs(want) + (2 * 2.0 ** -11 + 2 * score) * size + 2.0 ** -25
        tol += 80 * 2.0 ** -23 * 255 / 127 * np.abs(vh).max()
        err = np.abs(got[:, h].astype(np.float64) - want)
        assert np.isfinite(got[:, h]).all()
        worst = max(worst, float((err / tol).max()))
    assert worst <= 1, worst


def rows(seed, T, Hkv, D):
    rng = np.random.default_rng(seed)
    channel = np.exp(0.5 * rng.standard_normal((Hkv, D)))
    return [(rng.standard_normal((T, Hkv, D)) * channel).astype(np.float16) for _ in range(2)]


def queries(seed, n, H, D):
    return np.random.default_rng(seed + 1000).standard_normal((n, H, D)).astype(np.float16)


def same(a, b):
    return np.array_equal(np.asarray(a).view(np.uint16), np.asarray(b).view(np.uint16))


# ---- what the cache holds -------------------------------------------------------------------------------------

@pytest.mark.parametrize("Hkv,D", [(1, 128), (4, 64), (3, 128)])
@pytest.mark.parametrize("T", [1, 63, 64, 65, 130, 257])
def test_held_rows(dev, Hkv, D, T):
    """Rows come back as defined, whether they came as one prompt, in ragged pieces or one by one."""
    from tensorlogic_b200.api import KVCache8
    k, v = rows(T, T, Hkv, D)
    want = held_values(k), held_values(v)
    whole = KVCache8(dev, 2, Hkv, D, max_seq=T, max_batch=2)
    whole.append(1, dev.tensor(k), dev.tensor(v))
    pieces = KVCache8(dev, 1, Hkv, D, max_seq=300)
    at = 0
    for n in (1, 62, 2, 40, 100, 257):
        n = min(n, T - at)
        if n:
            pieces.append(0, dev.tensor(k[at:at + n]), dev.tensor(v[at:at + n]))
        at += n
    single = KVCache8(dev, 1, Hkv, D, max_seq=T, max_batch=3)
    for i in range(T):  # sequence 1 of three; the others stay empty
        single.append(0, dev.tensor(np.stack([k[i]] * 3)), dev.tensor(np.stack([v[i]] * 3)), positions=np.array([-1, i, -1]))
    for cache, layer, seq in ((whole, 1, 0), (pieces, 0, 0), (single, 0, 1)):
        got = cache.layer_arrays(layer, seq, T)
        assert same(got[0], want[0]) and same(got[1], want[1])
    assert not np.any(whole.layer_arrays(0, 0, T)[0]) and not np.any(whole.layer_arrays(1, 1, T)[1])  # nothing there
    assert not np.any(single.layer_arrays(0, 2, T)[0])
    assert list(single.lengths[0]) == [0, T, 0]
    dev.synchronize()


def test_held_rows_of_odd_values(dev):
    """Zeros, subnormals, values on a code's border, the largest f16, NaN and infinities."""
    from tensorlogic_b200.api import KVCache8
    Hkv, D = 8, 64
    k = np.random.default_rng(1).standard_normal((128, Hkv, D)).astype(np.float16)
    k[:64, 0] = 0
    k[:64, 1] = np.arange(64 * 64).reshape(64, 64) % 37 * 2.0 ** -24            # all subnormal
    k[:64, 2] = np.arange(64 * 64).reshape(64, 64) % 509 - 254                  # a = 254: odd values lie on borders
    k[:64, 3] = np.where(np.arange(64)[None, :] % 5, k[:64, 3], 65504)
    k[7, 4, 3], k[8, 4, 3], k[9, 4, 3] = np.nan, np.inf, -np.inf
    k[100, 5, 0], k[101, 5, 1], k[102, 5, 2] = np.nan, np.inf, -np.inf
    k[:64, 6] = 2.0 ** -24
    k[:64, 7] = -k[:64, 2]
    k[:64, 7, 0] = -0.0
    v = k[:, ::-1].copy()
    want = held_values(k), held_values(v)
    for n in (127, 128):  # the second block open, then sealed
        cache = KVCache8(dev, 1, Hkv, D, max_seq=128)
        cache.append(0, dev.tensor(k[:n]), dev.tensor(v[:n]))
        got = cache.layer_arrays(0)
        for g, x in zip(got, (k, v)):
            w = held_values(x[:n])
            assert np.array_equal(g, w) and np.isfinite(g).all()  # (-0 and 0 are one code)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("held,at,n", [(200, 100, 30), (200, 64, 1), (200, 0, 5), (128, 127, 1), (130, 70, 100), (70, 66, 3), (65, 1, 63)])
def test_rewind(dev, D, held, at, n):
    """Rows that join at an earlier position: those in front keep the values they were held as, the rest is gone."""
    from tensorlogic_b200.api import KVCache8
    k, v = rows(held, held, 2, D)
    k2, v2 = rows(held + 1, n, 2, D)
    cache = KVCache8(dev, 1, 2, D, max_seq=256)
    cache.append(0, dev.tensor(k), dev.tensor(v))
    for _ in range(2):  # a second time changes nothing
        cache.append(0, dev.tensor(k2), dev.tensor(v2), position=at)
        got = cache.layer_arrays(0, 0, 256)
        for g, old, new in zip(got, (k, v), (k2, v2)):
            sealed = held // BLOCK * BLOCK
            kept = np.concatenate([held_values(old)[:min(at, sealed)], old[min(at, sealed):at]])
            want = held_values(np.concatenate([kept, new]))
            assert same(g[:at + n], want) and not g[at + n:].any()
            # (a block whose values are codes already is sealed to the same values)
            assert same(held_values(held_values(old)), held_values(old))


def test_positions_outside_are_skipped_and_reported(dev):
    """Through the C interface a gap or a row past the end touches nothing; the next synchronize says so."""
    from tensorlogic_b200 import _lib
    from tensorlogic_b200.api import KVCache8, TensorError, _upload_i32
    k, v = rows(3, 70, 2, 64)
    cache = KVCache8(dev, 1, 2, 64, max_seq=70, max_batch=4)
    for s in range(4):
        cache.append(0, dev.tensor(k[:60 + s]), dev.tensor(v[:60 + s]), sequence=s)
    tk, tv = dev.tensor(k[:4]), dev.tensor(v[:4])
    pos = _upload_i32(dev, np.array([61, 61, 2**31 - 1, -5], np.int32))  # a gap; its end; far out; none
    _lib.check(dev.lib.tlc_kvcache8_append(dev.handle, cache.handle, 0, tk.ptr, tv.ptr, 4, 0, 0, pos.ptr))
    with pytest.raises(TensorError) as e:
        dev.synchronize()
    assert e.value.code == _lib.ERR_INDEX
    dev.synchronize()
    for s, new in enumerate((0, 1, 0, 0)):
        n = 60 + s
        x = np.concatenate([k[:n], k[s:s + 1]])[:n + new]
        got = cache.layer_arrays(0, s, 70)[0]
        assert same(got[:n + new], held_values(x)) and not got[n + new:].any()
    # a prompt in front of a gap
    _lib.check(dev.lib.tlc_kvcache8_append(dev.handle, cache.handle, 0, tk.ptr, tv.ptr, 4, 0, 66, None))
    with pytest.raises(TensorError):
        dev.synchronize()
    # queries whose keys are not there: they see what there is
    q = dev.tensor(queries(1, 4, 2, 64))
    out = dev.empty((4, 2, 64))
    pos = _upload_i32(dev, np.array([59, 2**31 - 1, -2**31, 62], np.int32))
    _lib.check(dev.lib.tlc_attention8(dev.handle, cache.handle, 0, q.ptr, out.ptr, 4, 1, 2, 0, 0, pos.ptr, 70, 0.125))
    with pytest.raises(TensorError) as e:
        dev.synchronize()
    assert e.value.code == _lib.ERR_INDEX
    got = out.numpy()
    qh = queries(1, 4, 2, 64)
    for s, n in ((0, 60), (1, 62), (3, 63)):
        x = np.concatenate([k[:60 + s], k[s:s + 1]]) if s == 1 else k[:60 + s]
        y = np.concatenate([v[:60 + s], v[s:s + 1]]) if s == 1 else v[:60 + s]
        check_attention(got[s:s + 1], qh[s:s + 1], exact_values(x), exact_values(y), n - 1, 0.125)
    assert not got[2].any()
    dev.synchronize()


# ---- attention ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("H,Hkv,D", [(32, 4, 64), (8, 1, 128), (4, 4, 64), (6, 2, 128), (20, 1, 64), (12, 1, 128)])
@pytest.mark.parametrize("T", [1, 2, 63, 64, 65, 129, 641, 2048])
def test_decode(dev, H, Hkv, D, T):
    from tensorlogic_b200.api import KVCache8
    k, v = rows(T + H, T, Hkv, D)
    q = queries(T, 1, H, D)
    cache = KVCache8(dev, 2, Hkv, D, max_seq=2048)
    cache.append(1, dev.tensor(k), dev.tensor(v))
    ek, ev = exact_values(k), exact_values(v)
    by_position = cache.attention(1, dev.tensor(q), H, positions=np.array([T - 1])).numpy()
    check_attention(by_position, q, ek, ev, T - 1)
    check_attention(cache.attention(1, dev.tensor(q), H, q_pos0=T - 1).numpy(), q, ek, ev, T - 1)
    if T > 70:  # an earlier position: sealed blocks of which it sees a part
        check_attention(cache.attention(1, dev.tensor(q), H, positions=np.array([T - 70])).numpy(), q, ek, ev, T - 70)
    dev.synchronize()


@pytest.mark.parametrize("H,Hkv,D,T", [(8, 1, 64, 20000), (32, 4, 64, 9001), (8, 2, 128, 16383)])
def test_decode_long_context(dev, H, Hkv, D, T):
    """Keys shared out over many CTAs; the launch is sized by the cache, not by the position, where that is far off."""
    from tensorlogic_b200 import _lib
    from tensorlogic_b200.api import KVCache8, _upload_i32
    k, v = rows(T, T, Hkv, D)
    k[T // 2] *= 4  # some keys count more than others
    q = queries(T, 1, H, D)
    cache = KVCache8(dev, 1, Hkv, D, max_seq=32768)
    for at in range(0, T, 5000):
        cache.append(0, dev.tensor(k[at:at + 5000]), dev.tensor(v[at:at + 5000]))
    ek, ev = exact_values(k), exact_values(v)
    for pos in (T - 1, 100):
        check_attention(cache.attention(0, dev.tensor(q), H, positions=np.array([pos])).numpy(), q, ek, ev, pos)
        tq, tp, out = dev.tensor(q), _upload_i32(dev, np.array([pos], np.int32)), dev.empty(q.shape)
        _lib.check(dev.lib.tlc_attention8(dev.handle, cache.handle, 0, tq.ptr, out.ptr, 1, 1, H, 0, 0, tp.ptr, 32768, D ** -0.5))
        check_attention(out.numpy(), q, ek, ev, pos)
    dev.synchronize()


@pytest.mark.parametrize("H,Hkv,D,batch,T", [(32, 4, 64, 5, 500), (8, 8, 128, 33, 200), (8, 1, 128, 8, 1100)])
def test_decode_ragged_batch(dev, H, Hkv, D, batch, T):
    """Sequences of different lengths, an idle slot; rows behind the batch stay as they were."""
    from tensorlogic_b200 import _lib
    from tensorlogic_b200.api import KVCache8, _upload_i32
    lengths = [max(1, T - 37 * i) for i in range(batch)]
    data = [rows(10 * b + 1, n, Hkv, D) for b, n in enumerate(lengths)]
    cache = KVCache8(dev, 1, Hkv, D, max_seq=T, max_batch=batch + 2)
    for b, (k, v) in enumerate(data):
        cache.append(0, dev.tensor(k), dev.tensor(v), sequence=b + 1)  # sequences 1 ..
    q = queries(5, batch, H, D)
    pos = np.array([n - 1 for n in lengths], np.int32)
    pos[2] = -1
    mark = np.full((batch + 1, H, D), 7, np.float16)
    out, tq, tp = dev.tensor(mark), dev.tensor(q), _upload_i32(dev, pos)
    _lib.check(dev.lib.tlc_attention8(dev.handle, cache.handle, 0, tq.ptr, out.ptr, batch, 1, H, 1, 0, tp.ptr, T, D ** -0.5))
    got = out.numpy()
    assert same(got[batch], mark[batch]) and not got[2].any()
    for b, (k, v) in enumerate(data):
        if b != 2:
            check_attention(got[b:b + 1], q[b:b + 1], exact_values(k), exact_values(v), lengths[b] - 1)
    assert same(cache.attention(0, tq, H, positions=pos, batch=batch, sequence=1).numpy(), got[:batch])
    dev.synchronize()


@pytest.mark.parametrize("H,Hkv,D", [(32, 4, 64), (4, 4, 128), (6, 2, 64), (20, 1, 128)])
@pytest.mark.parametrize("I,pos0", [(2, 0), (17, 0), (64, 0), (77, 391), (130, 62), (300, 5), (3, 1000)])
def test_prefill(dev, H, Hkv, D, I, pos0):
    from tensorlogic_b200.api import KVCache8
    k, v = rows(I + pos0, pos0 + I, Hkv, D)
    q = queries(I, I, H, D)
    cache = KVCache8(dev, 1, Hkv, D, max_seq=pos0 + I + 3, max_batch=2)
    cache.append(0, dev.tensor(k), dev.tensor(v), sequence=1)
    got = cache.attention(0, dev.tensor(q), H, q_pos0=pos0, sequence=1).numpy()
    check_attention(got, q, exact_values(k), exact_values(v), pos0)
    dev.synchronize()


def test_prefill_of_a_document(dev):
    """Long enough for every tile to be full; a second sequence of the same batch."""
    from tensorlogic_b200.api import KVCache8
    H, Hkv, D, I = 8, 2, 128, 1100
    cache = KVCache8(dev, 1, Hkv, D, max_seq=I, max_batch=2)
    data = [rows(b, I, Hkv, D) for b in range(2)]
    for b, (k, v) in enumerate(data):
        cache.append(0, dev.tensor(k), dev.tensor(v), sequence=b)
    q = queries(9, 2 * I, H, D)
    got = cache.attention(0, dev.tensor(q), H, batch=2).numpy()
    for b, (k, v) in enumerate(data):
        check_attention(got[b * I:(b + 1) * I], q[b * I:(b + 1) * I], exact_values(k), exact_values(v), 0)
    dev.synchronize()


@pytest.mark.parametrize("I,T", [(40, 60), (40, 100), (300, 300), (700, 700)])
def test_masked_keys_do_not_matter(dev, I, T):
    """Keys and values behind a query, NaN and infinities among them, change nothing in its row; nor does what a block held
    before it was rewound."""
    from tensorlogic_b200.api import KVCache8
    H, Hkv, D = 8, 1, 64
    k, v = rows(T, T, Hkv, D)
    q = queries(T, I, H, D)
    clean = KVCache8(dev, 1, Hkv, D, max_seq=T)
    clean.append(0, dev.tensor(k), dev.tensor(v))
    want = clean.attention(0, dev.tensor(q), H, q_pos0=T - I).numpy()
    bad_k, bad_v = k.copy(), v.copy()
    bad_k[T - 1], bad_v[T - 1] = np.nan, np.inf
    other = KVCache8(dev, 1, Hkv, D, max_seq=T)
    other.append(0, dev.tensor(bad_k), dev.tensor(bad_v))
    got = other.attention(0, dev.tensor(q), H, q_pos0=T - I).numpy()
    check_attention(got, q, exact_values(bad_k), exact_values(bad_v), T - I)
    if T % BLOCK:  # (in a sealed block the last row changes the others' codes)
        assert same(got[:-1], want[:-1])
    other.append(0, dev.tensor(k), dev.tensor(v), position=0)
    assert same(other.attention(0, dev.tensor(q), H, q_pos0=T - I).numpy(), want)


def test_extreme_values(dev):
    """The largest f16 in keys, values and scale factors; blocks of very different size side by side."""
    from tensorlogic_b200.api import KVCache8
    H, Hkv, D, T = 4, 1, 64, 200
    k, v = rows(1, T, Hkv, D)
    k[:64] *= 2.0 ** -10
    v[:64] *= 2.0 ** -12
    v[64:128] = np.where(v[64:128] > 0, 65504, -65504)
    k[70, 0, :] = 30
    q = queries(2, T, H, D)
    cache = KVCache8(dev, 1, Hkv, D, max_seq=T)
    cache.append(0, dev.tensor(k), dev.tensor(v))
    for scale in (None, 0.0, -0.125, 2.0):
        got = cache.attention(0, dev.tensor(q), H, scale=scale).numpy()
        check_attention(got, q, exact_values(k), exact_values(v), 0, scale)
        got = cache.attention(0, dev.tensor(q[T - 1:]), H, q_pos0=T - 1, scale=scale).numpy()
        check_attention(got, q[T - 1:], exact_values(k), exact_values(v), T - 1, scale)


def test_two_calls_are_the_same(dev):
    """Shared keys are joined in a fixed order: the same call gives the same bits."""
    from tensorlogic_b200.api import KVCache8
    k, v = rows(1, 9000, 1, 128)
    q = dev.tensor(queries(1, 1, 8, 128))
    cache = KVCache8(dev, 1, 1, 128, max_seq=9000)
    cache.append(0, dev.tensor(k), dev.tensor(v))
    first = cache.attention(0, q, 8, q_pos0=8999).numpy()
    for _ in range(5):
        assert same(cache.attention(0, q, 8, q_pos0=8999).numpy(), first)


def test_captured_step(dev):
    """Append and attention of a decode step in a graph: replays follow the positions on the device."""
    import torch
    from tensorlogic_b200 import _lib
    from tensorlogic_b200.api import KVCache8
    H, Hkv, D, B, T = 8, 2, 64, 3, 150
    data = [rows(b, T, Hkv, D) for b in range(B)]
    q = queries(1, B, H, D)
    eager, graph = (KVCache8(dev, 1, Hkv, D, max_seq=T, max_batch=B) for _ in range(2))
    start = [60, 0, 127]
    for c in (eager, graph):
        for b in range(B):
            if start[b]:
                c.append(0, dev.tensor(data[b][0][:start[b]]), dev.tensor(data[b][1][:start[b]]), sequence=b)
    dev.synchronize()
    tk, tv = (torch.empty(B, Hkv, D, dtype=torch.float16, device="cuda") for _ in range(2))
    tq, out = torch.tensor(q, device="cuda"), torch.empty(B, H, D, dtype=torch.float16, device="cuda")
    pos = torch.empty(B, dtype=torch.int32, device="cuda")

    def step(cache):
        _lib.check(dev.lib.tlc_kvcache8_append(dev.handle, cache.handle, 0, tk.data_ptr(), tv.data_ptr(), B, 0, 0, pos.data_ptr()))
        _lib.check(dev.lib.tlc_attention8(dev.handle, cache.handle, 0, tq.data_ptr(), out.data_ptr(), B, 1, H, 0, 0, pos.data_ptr(), T, 0.125))

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(dev.stream)):
        step(graph)
    for i in range(10):
        for b in range(B):
            tk[b].copy_(torch.tensor(data[b][0][start[b] + i]))
            tv[b].copy_(torch.tensor(data[b][1][start[b] + i]))
        pos.copy_(torch.tensor([s + i for s in start], dtype=torch.int32))
        torch.cuda.synchronize()
        step(eager)
        dev.synchronize()
        want = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        for b in range(B):
            n = start[b] + i + 1
            check_attention(out[b:b + 1].cpu().numpy(), q[b:b + 1], exact_values(data[b][0][:n]), exact_values(data[b][1][:n]), n - 1)
    dev.synchronize()


def test_refusals(dev):
    from tensorlogic_b200 import _lib
    from tensorlogic_b200.api import Device, KVCache8, TensorError
    for args in ((1, 2, 96), (1, 2, 0), (0, 2, 64), (1, 0, 64)):
        with pytest.raises(TensorError):
            KVCache8(dev, *args)
    cache = KVCache8(dev, 2, 2, 64, max_seq=100, max_batch=2)
    t = dev.empty((4, 2, 64))
    lib, h, c = dev.lib, dev.handle, cache.handle

    def append(layer=0, k=t.ptr, v=t.ptr, m=1, seq=0, at=0, pos=None, ctx=h, cache=c):
        return lib.tlc_kvcache8_append(ctx, cache, layer, k, v, m, seq, at, pos)

    def attend(layer=0, q=t.ptr, out=t.ptr, batch=1, n=1, heads=2, seq=0, at=0, pos=None, most=0, ctx=h, cache=c):
        return lib.tlc_attention8(ctx, cache, layer, q, out, batch, n, heads, seq, at, pos, most, 0.125)

    def read(layer=0, seq=0, n_seq=1, first=0, n=1, k=t.ptr, v=t.ptr, ctx=h, cache=c):
        return lib.tlc_kvcache8_rows(ctx, cache, layer, seq, n_seq, first, n, k, v)

    bad, index, shape, dim = _lib.ERR_INVALID_OPERATION, _lib.ERR_INDEX, _lib.ERR_SHAPE_MISMATCH, _lib.ERR_INVALID_DIMENSION
    assert append(k=None) == bad and append(v=t.ptr + 2) == bad and append(cache=None) == bad and append(m=-1) == dim
    assert append(layer=2) == index and append(layer=-1) == index and append(at=100) == index and append(at=-1) == index
    assert append(m=2**31 - 1, at=5) == index and append(seq=2) == shape and append(seq=-1) == shape
    assert append(m=3, pos=t.ptr) == shape and append(m=2, seq=1, pos=t.ptr) == shape
    assert append(m=0) == 0
    assert attend(q=None) == bad and attend(out=t.ptr + 8) == bad and attend(batch=0) == shape and attend(batch=3) == shape
    assert attend(layer=2) == index and attend(heads=3) == shape and attend(heads=0) == shape and attend(n=0) == bad
    assert attend(n=101) == index and attend(at=100) == index and attend(at=-1) == index and attend(at=2**31 - 1) == index
    assert attend(pos=t.ptr, n=2, most=5) == bad and attend(pos=t.ptr, most=101) == index and attend(pos=t.ptr, most=0) == index
    assert read(k=None) == bad and read(n=101) == index and read(first=2**31 - 1) == index and read(n_seq=3) == shape
    assert read(n=-1) == index and read(n=0) == 0 and read(v=t.ptr + 2) == bad
    other = Device(0)  # another context, that is another stream: the cache's workspace serves one
    try:
        assert append(ctx=other.handle) == _lib.ERR_DEVICE and attend(ctx=other.handle) == _lib.ERR_DEVICE
        assert read(ctx=other.handle) == _lib.ERR_DEVICE
    finally:
        other.close()
    dev.synchronize()


@pytest.mark.parametrize("prepared", [False, True])
def test_captured_prompt(dev, prepared):
    """A long prompt in a graph: with what its fast kernel keeps made before, and without, where nothing may be made."""
    import torch
    from tensorlogic_b200 import _lib
    from tensorlogic_b200.api import KVCache8
    H, Hkv, D, I = 8, 2, 128, 900
    k, v = rows(2, I, Hkv, D)
    q = queries(2, I, H, D)
    cache = KVCache8(dev, 1, Hkv, D, max_seq=1000, max_batch=2)
    cache.append(0, dev.tensor(k), dev.tensor(v), sequence=1)
    first = cache.attention(0, dev.tensor(q), H, sequence=1).numpy() if prepared else None
    tq, out = torch.tensor(q, device="cuda"), torch.zeros(I, H, D, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(dev.stream)):
        _lib.check(dev.lib.tlc_attention8(dev.handle, cache.handle, 0, tq.data_ptr(), out.data_ptr(), 1, I, H, 1, 0, None, 0, D ** -0.5))
    g.replay()
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    check_attention(got, q, exact_values(k), exact_values(v), 0)
    assert not prepared or same(got, first)
    dev.synchronize()


def test_far_into_memory(dev):
    """The last sequence of the last layer of a cache of more than 2^32 bytes."""
    from tensorlogic_b200.api import KVCache8
    H, Hkv, D, B, T = 16, 8, 128, 40, 777
    cache = KVCache8(dev, 2, Hkv, D, max_seq=32768, max_batch=B)
    k, v = rows(3, T, Hkv, D)
    q = queries(3, T, H, D)
    cache.append(1, dev.tensor(k[:-1]), dev.tensor(v[:-1]), sequence=B - 1)
    pos = np.array([-1, T - 1])
    cache.append(1, dev.tensor(np.stack([k[-1]] * 2)), dev.tensor(np.stack([v[-1]] * 2)), positions=pos, sequence=B - 2)
    got = cache.layer_arrays(1, B - 1)
    assert same(got[0], held_values(k)) and same(got[1], held_values(v))
    assert not np.any(cache.layer_arrays(1, B - 2, 5)[0])
    prompt = cache.attention(1, dev.tensor(q), H, sequence=B - 1).numpy()
    token = cache.attention(1, dev.tensor(q[-2:]), H, batch=2, positions=pos, sequence=B - 2).numpy()
    check_attention(prompt, q, exact_values(k), exact_values(v), 0)
    check_attention(token[1:], q[-1:], exact_values(k), exact_values(v), T - 1)
    assert not token[0].any()
    dev.synchronize()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("I", [1, 8, 400])
def test_scales_apart(dev, D, I):
    """Blocks of very different scale, and in a block of large values one row of tiny ones that most of P falls on."""
    from tensorlogic_b200.api import KVCache8
    H, Hkv, T = 4, 2, 640
    k, v = (a.astype(np.float32) for a in rows(7, T, Hkv, D))
    for a in (k, v):
        a[:64] *= 30
        a[64:320] *= 1e-3
    q = queries(7, I, H, D)
    k[5] = 8 * q[0].reshape(Hkv, H // Hkv, D)[:, 0] / np.sqrt(D) * 8
    v[5] = 1e-4
    k, v = k.astype(np.float16), v.astype(np.float16)
    cache = KVCache8(dev, 1, Hkv, D, max_seq=T)
    cache.append(0, dev.tensor(k), dev.tensor(v))
    got = cache.attention(0, dev.tensor(q), H, q_pos0=T - I).numpy()
    check_attention(got, q, exact_values(k), exact_values(v), T - I)
