"""The operators around an 8-bit KV cache and the log probabilities of tokens, as measurable cases.

  append     rows of K and V into the cache, a prompt's or one a sequence (``tlc_kvcache8_append``), and the cache
             rows of the blocks they fall into read back (``tlc_kvcache8_rows``)
  decode     attention of one query a sequence over that cache (``tlc_attention8`` with positions on the device)
  prefill    attention of a prompt's queries over it (``tlc_attention8``)
  logprobs   log probabilities of given tokens, entropy and the likeliest alternatives (``tlc_token_logprobs``)

The cache holds blocks of 64 positions of a KV head as 8-bit codes with one scale, rint(127 x / a) and a / 127 for a
block whose largest magnitude is a; the rows of a block that is not full are kept as they came, in f16.

``own`` is set by whoever runs the cases: false computes the operators from elementary torch operations, true calls the
package.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 64
# Query heads, KV heads, head size: the benchmark's model shapes; the last is what one of eight GPUs holds of the 70B.
HEADS = {"tinyllama": (32, 4, 64), "llama2_7b": (32, 32, 128), "llama2_70b_rank_of_8": (8, 1, 128)}


def listed():
    return [
        # A decode step of a full batch: 32 chats of different lengths, a token each; some fill their block.
        dict(name="append_tiny_b32", kind="append", model="tinyllama", batch=32, rows=1, pos0=767, gap=3),
        # A further turn of a chat: a ragged prompt that starts and ends within a block.
        dict(name="append_tiny_77_turn", kind="append", model="tinyllama", batch=1, rows=77, pos0=391, gap=0),
        # A long document into the 7B shape.
        dict(name="append_7b_2048", kind="append", model="llama2_7b", batch=1, rows=2048, pos0=0, gap=0),
        # One chat with the small model: the smallest call.
        dict(name="decode_tiny_b1_512", kind="decode", model="tinyllama", batch=1, context=512, gap=0),
        # A served 7B model, a full batch of ragged contexts: what the cache's bytes bound.
        dict(name="decode_7b_b32_768", kind="decode", model="llama2_7b", batch=32, context=768, gap=11),
        # One GPU's share of the 70B shape, eight long contexts over its one KV head.
        dict(name="decode_70b_rank_b8_2048", kind="decode", model="llama2_70b_rank_of_8", batch=8, context=2048, gap=0),
        # One very long context over few heads: keys have to be shared out over the whole GPU.
        dict(name="decode_tiny_b1_65000", kind="decode", model="tinyllama", batch=1, context=65000, gap=0),
        # The queries of that further turn.
        dict(name="prefill_tiny_77_turn", kind="prefill", model="tinyllama", rows=77, pos0=391),
        # The queries of that document: the most work.
        dict(name="prefill_7b_2048", kind="prefill", model="llama2_7b", rows=2048, pos0=0),
        # The token just sampled, with five alternatives: what a chat API returns with each token.
        dict(name="logprobs_1x32000_top5", kind="logprobs", rows=1, vocab=32000, top=5, masked=0.0),
        # Scoring a prompt of 512 tokens (perplexity): no alternatives.
        dict(name="logprobs_512x32000", kind="logprobs", rows=512, vocab=32000, top=0, masked=0.0),
        # A batch with a large vocabulary of odd size, a grammar's mask, twenty alternatives.
        dict(name="logprobs_37x100003_top20", kind="logprobs", rows=37, vocab=100003, top=20, masked=0.3),
    ]


def _log(rng, lo, hi):
    """A size between lo and hi, even in its logarithm."""
    return max(int(lo), min(int(hi), int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "decode", "decode", "prefill", "logprobs"))
    model = rng.choice(tuple(HEADS))
    row = HEADS[model][1] * HEADS[model][2]
    if kind == "append":
        if rng.random() < 0.5:  # a token a sequence
            batch = _log(rng, 1, 32)
            pos0 = _log(rng, 1, 2047)
            return dict(kind=kind, model=model, batch=batch, rows=1, pos0=pos0, gap=rng.randint(0, min(3, pos0 // batch)))
        rows = _log(rng, 1, 2048)
        return dict(kind=kind, model=model, batch=1, rows=rows, pos0=rng.choice((0, rng.randint(0, 2048 - rows))), gap=0)
    if kind == "decode":
        batch = _log(rng, 1, 32)
        context = _log(rng, 1, min(65536, 24576 * 4096 // (batch * row)))
        return dict(kind=kind, model=model, batch=batch, context=context, gap=rng.randint(0, context // (2 * batch)))
    if kind == "prefill":
        rows = _log(rng, 2, 2048)
        return dict(kind=kind, model=model, rows=rows, pos0=rng.choice((0, rng.randint(0, 2048 - rows))))
    vocab = _log(rng, 1000, 160000)
    return dict(kind=kind, rows=_log(rng, 1, min(2048, 16384000 // vocab)), vocab=vocab, top=rng.choice((0, 1, 5, 20, 32)),
                masked=rng.choice((0.0, 0.0, 0.3, 0.99)))


# ---- inputs -------------------------------------------------------------------------------------------------

def _generator(seed, tag):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1009 + tag)
    return g


def _rows(seed, tag, *shape):
    """Rows of K or V as projections give them, f16 [..., heads, size]: normal, with channels of different size."""
    g = _generator(seed, tag)
    channel = torch.exp(0.5 * torch.randn(shape[-2:], generator=g, device="cuda"))
    return (torch.randn(shape, generator=g, device="cuda") * channel).half()


def _inputs(case, seed):
    """The data of a case, the same for both forms: contexts and new rows, queries, positions, logits."""
    if case["kind"] == "logprobs":
        g = _generator(seed, 1)
        rows, vocab = case["rows"], case["vocab"]
        spread = 1.0 + 2.0 * torch.rand(rows, 1, generator=g, device="cuda")  # sure and unsure rows
        logits = (torch.randn(rows, vocab, generator=g, device="cuda") * spread).half()
        if case["masked"]:
            logits[torch.rand(rows, vocab, generator=g, device="cuda") < case["masked"]] = -math.inf
        targets = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        greedy = torch.rand(rows, generator=g, device="cuda") < 0.5
        return dict(logits=logits, targets=torch.where(greedy, logits.float().argmax(1), targets).int())
    H, kv, D = HEADS[case["model"]]
    batch = case.get("batch", 1)
    if case["kind"] == "decode":  # the query's own key is the newest in the cache
        pos = [case["context"] - 1 - case["gap"] * i for i in range(batch)]
        held, rows = [p + 1 for p in pos], 1
    elif case["kind"] == "prefill":
        pos, rows = [case["pos0"]], case["rows"]
        held = [case["pos0"] + rows]
    else:
        pos, rows = [case["pos0"] - case["gap"] * i for i in range(batch)], case["rows"]
        held = pos
    d = dict(pos=pos, held=held, positions=torch.tensor(pos, dtype=torch.int32, device="cuda"))
    d["k"], d["v"] = (_rows(seed, t, batch, max(held), kv, D) for t in (1, 2))
    if case["kind"] == "append":
        d["new_k"], d["new_v"] = (_rows(seed, t, batch, rows, kv, D) for t in (3, 4))
        last = max(p + rows for p in pos)
        d["window"] = (min(pos) // BLOCK * BLOCK, last)
    else:
        d["q"] = torch.randn(batch * rows, H, D, generator=_generator(seed, 5), device="cuda").half()
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    s = dict(case=case)
    if case["kind"] == "logprobs":
        rows, top = case["rows"], case["top"]
        s.update(d)
        if own:
            s["dev"] = _device()
            s["out"] = [torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"),
                        torch.empty(rows, top, dtype=torch.int32, device="cuda"), torch.empty(rows, top, device="cuda")]
        return s
    kv, D = HEADS[case["model"]][1:]
    s.update({n: d[n] for n in ("q", "new_k", "new_v", "pos", "positions", "window") if n in d})
    batch, held = len(d["pos"]), d["held"]
    if own:
        from tensorlogic_b200.api import KVCache8
        s["dev"] = _device()
        s["cache"] = KVCache8(s["dev"], 1, kv, D, max_seq=max(p + case.get("rows", 1) for p in d["pos"]), max_batch=batch)
        torch.cuda.synchronize()  # the library has a stream of its own
        for b in range(batch):
            if held[b]:
                _append(s, d["k"][b], d["v"][b], held[b], b, 0, None)
        if case["kind"] == "append":
            shape = (batch, s["window"][1] - s["window"][0], kv, D)
            s["out"] = [torch.empty(shape, dtype=torch.float16, device="cuda") for _ in range(2)]
        else:
            s["out"] = torch.empty_like(s["q"])
        s["dev"].synchronize()
        return s
    # The plain form's cache: codes and scales of the full blocks, and each sequence's newest rows in f16.
    full = torch.tensor([h // BLOCK for h in held], device="cuda")
    s["full"] = full
    nb = max(held) // BLOCK
    s["cache"] = []
    for x in (d["k"], d["v"]):
        codes, scale = _quantize(x[:, : nb * BLOCK].unflatten(1, (nb, BLOCK)))
        newest = torch.zeros(batch, BLOCK, kv, D, dtype=torch.float16, device="cuda")
        at = full[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")
        there = at < torch.tensor(held, device="cuda")[:, None]
        rows = torch.arange(batch, device="cuda")[:, None].expand_as(at)
        newest[there] = x[rows[there], at[there]]
        s["cache"].append((codes, scale, newest))
    return s


# ---- the plain form -----------------------------------------------------------------------------------------

def _quantize(x):
    """Codes and scales of blocks [..., block, 64, heads, size]."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=65504.0, neginf=-65504.0)
    a = x.abs().amax((-3, -1), keepdim=True)
    return torch.where(a > 0, torch.round(127 * x / a), 0.0).to(torch.int8), a / 127


def _values(part, full, blocks):
    """What the cache holds of positions 0 .. 64 blocks, f32 [batch, position, heads, size]; zeros past its rows."""
    codes, scale, newest = part
    x = codes.float() * scale
    batch, nb = x.shape[:2]
    x = torch.cat([x, x.new_zeros(batch, blocks + 1 - nb, *x.shape[2:])], 1).flatten(1, 2)
    at = full[:, None] * BLOCK + torch.arange(BLOCK, device=x.device)
    x[torch.arange(batch, device=x.device)[:, None], at] = newest.float()
    return x[:, : blocks * BLOCK]


def _plain_append(s):
    lo, hi = s["window"]
    blocks = -(-hi // BLOCK)
    pos, rows = s["positions"].long(), s["new_k"].shape[1]
    out = []
    for part, new in zip(s["cache"], (s["new_k"], s["new_v"])):
        x = _values(part, s["full"], blocks)
        at = pos[:, None] + torch.arange(rows, device=x.device)
        x[torch.arange(x.shape[0], device=x.device)[:, None], at] = new.float()
        x = x[:, lo:].unflatten(1, (-1, BLOCK))
        codes, scale = _quantize(x)
        block = torch.arange(lo // BLOCK, blocks, device=x.device)
        done = (block >= pos[:, None] // BLOCK) & (block < (pos[:, None] + rows) // BLOCK)  # filled by this call
        x = torch.where(done[..., None, None, None], codes.float() * scale, x).flatten(1, 2)
        there = torch.arange(lo, blocks * BLOCK, device=x.device) < pos[:, None] + rows
        out.append(torch.where(there[..., None, None], x, 0.0)[:, : hi - lo].half())
    return out


def _plain_attention(s):
    case = s["case"]
    H, kv, D = HEADS[case["model"]]
    batch, rows = len(s["pos"]), case.get("rows", 1)
    last = max(s["pos"]) + rows
    k, v = (_values(part, s["full"], -(-last // BLOCK))[:, :last] for part in s["cache"])
    q = s["q"].float().view(batch, rows, kv, H // kv, D)
    scores = torch.einsum("bihgd,bthd->bhgit", q, k) / math.sqrt(D)
    at = s["positions"].long()[:, None] + torch.arange(rows, device=k.device)
    hidden = torch.arange(last, device=k.device) > at[..., None]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    p = scores.exp_()
    out = torch.einsum("bhgit,bthd->bihgd", p, v) / p.sum(-1).permute(0, 3, 1, 2)[..., None]
    return out.reshape(batch * rows, H, D).half()


def _plain_logprobs(s):
    x, top = s["logits"].float(), s["case"]["top"]
    there = torch.isfinite(x)
    x = torch.where(there, x, -math.inf)
    m = x.amax(1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(1, keepdim=True)
    norm = m + total.log()
    entropy = norm - (torch.where(there, x, 0.0) * e).sum(1, keepdim=True) / total
    best, ids = torch.sort(x, dim=1, descending=True, stable=True) if top else (x, s["targets"].long()[:, None])
    best, ids = best[:, :top], torch.where(best[:, :top] == -math.inf, -1, ids[:, :top])
    return [(x.gather(1, s["targets"].long()[:, None]) - norm)[:, 0], entropy[:, 0], ids.int(), best - norm]


# ---- one pass -----------------------------------------------------------------------------------------------

_dev = None


def _device():
    global _dev
    if _dev is None:
        from tensorlogic_b200.api import Device
        _dev = Device()
    return _dev


def _check(rc):
    if rc:
        from tensorlogic_b200 import _lib
        _lib.check(rc)


def _append(s, k, v, rows, sequence, pos, positions):
    dev = s["dev"]
    _check(dev.lib.tlc_kvcache8_append(dev.handle, s["cache"].handle, 0, k.data_ptr(), v.data_ptr(), rows, sequence, pos,
                                       positions))


def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if not own:
        return {"append": _plain_append, "logprobs": _plain_logprobs}.get(kind, _plain_attention)(s)
    dev = s["dev"]
    if kind == "logprobs":
        lp, entropy, ids, top = s["out"]
        k = case["top"]
        _check(dev.lib.tlc_token_logprobs(dev.handle, s["logits"].data_ptr(), case["rows"], case["vocab"],
                                          s["targets"].data_ptr(), k, lp.data_ptr(), entropy.data_ptr(),
                                          ids.data_ptr() if k else None, top.data_ptr() if k else None))
        return s["out"]
    batch = len(s["pos"])
    if kind == "append":
        if case["rows"] == 1:  # a row for each sequence, its position on the device
            _append(s, s["new_k"], s["new_v"], batch, 0, 0, s["positions"].data_ptr())
        else:
            _append(s, s["new_k"], s["new_v"], case["rows"], 0, case["pos0"], None)
        (lo, hi), (k, v) = s["window"], s["out"]
        _check(dev.lib.tlc_kvcache8_rows(dev.handle, s["cache"].handle, 0, 0, batch, lo, hi - lo, k.data_ptr(), v.data_ptr()))
        return s["out"]
    H, _, D = HEADS[case["model"]]
    q, out, decode = s["q"], s["out"], kind == "decode"
    _check(dev.lib.tlc_attention8(dev.handle, s["cache"].handle, 0, q.data_ptr(), out.data_ptr(), batch,
                                  1 if decode else case["rows"], H, 0, 0 if decode else case["pos0"],
                                  s["positions"].data_ptr() if decode else None, max(s["pos"]) + 1 if decode else 0,
                                  1.0 / math.sqrt(D)))
    return out


# ---- what a pass cannot do without, and its outputs in 64 bits ------------------------------------------------

def work(case):
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": 2.0 * n + case["rows"] * (12 + 8 * case["top"]), "flops": 6.0 * n}
    H, kv, D = HEADS[case["model"]]
    row = kv * D
    if case["kind"] == "append":
        m, b = case["rows"], case["batch"]
        lo = (case["pos0"] - case["gap"] * (b - 1)) // BLOCK * BLOCK
        window = (case["pos0"] + m - lo) * b
        # new rows in, stored once (a byte a value when their block is full), the window read and handed back in f16
        full = m / BLOCK if m > 1 else b / BLOCK
        stored = row * 2 * (full * BLOCK + 2 * min(BLOCK / 2, m) * b)
        return {"bytes": 4.0 * row * m * b + stored + window * row * 2 * (1 + 2), "flops": 8.0 * window * row}
    if case["kind"] == "decode":
        keys = sum(case["context"] - case["gap"] * i for i in range(case["batch"]))
        return {"bytes": 2.0 * row * keys + 4.0 * case["batch"] * H * D, "flops": 4.0 * H * D * keys}
    n, p = case["rows"], case["pos0"]
    return {"bytes": 2.0 * row * (p + n) + 4.0 * n * H * D, "flops": 4.0 * H * D * (n * p + n * (n + 1) / 2)}


def _exact_rows(x, held):
    """What the cache holds of one sequence's rows [T, heads, size] given one after another, in 64 bits."""
    x = x[:held].double()
    n = held // BLOCK * BLOCK
    if n:
        y = x[:n].reshape(-1, BLOCK, *x.shape[1:])
        a = y.abs().amax((1, 3), keepdim=True)
        x[:n] = (torch.round(127 * y / a) * a / 127).reshape(n, *x.shape[1:])
    return x


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "logprobs":
        lp, entropy, ids, best = [], [], [], []
        for row, t in zip(d["logits"].double(), d["targets"].tolist()):
            at = torch.nonzero(torch.isfinite(row))[:, 0]
            x = row[at]
            logp = x - torch.logsumexp(x, 0)
            whole = torch.full_like(row, -math.inf)
            whole[at] = logp
            lp.append(whole[t])
            entropy.append(-(logp.exp() * logp).sum())
            order = torch.sort(x, descending=True, stable=True).indices[: case["top"]]
            pad = case["top"] - order.numel()
            ids.append(torch.cat([at[order], at.new_full((pad,), -1)]).int())
            best.append(torch.cat([logp[order], logp.new_full((pad,), -math.inf)]))
        return [torch.stack(lp), torch.stack(entropy), torch.stack(ids), torch.stack(best)]
    H, kv, D = HEADS[case["model"]]
    rows = case.get("rows", 1)
    if case["kind"] == "append":
        lo, hi = d["window"]
        out = []
        for old, new in ((d["k"], d["new_k"]), (d["v"], d["new_v"])):
            seqs = []
            for b, p in enumerate(d["pos"]):
                held = _exact_rows(torch.cat([old[b, :p], new[b]]), p + rows)
                seqs.append(torch.cat([held, held.new_zeros(max(0, hi - p - rows), kv, D)])[lo:hi])
            out.append(torch.stack(seqs))
        return out
    out = []
    for b, p in enumerate(d["pos"]):
        k, v = (_exact_rows(d[n][b], d["held"][b]) for n in ("k", "v"))
        q = d["q"].double().view(len(d["pos"]), rows, H, D)[b]
        heads = []
        for h in range(H):
            x = q[:, h] @ k[:, h // (H // kv)].T * D ** -0.5
            x = x.masked_fill(torch.arange(k.shape[0], device=x.device) > p + torch.arange(rows, device=x.device)[:, None], -math.inf)
            heads.append(torch.softmax(x, 1) @ v[:, h // (H // kv)])
        out.append(torch.stack(heads, 1))
    return torch.cat(out)
