"""Operator cases: attention over the states of what a search found, and the training of what made them.

Three operators, reached through veckern_amd.attention:

  attend            attention of query tokens to an encoder's states of another length, held as rows of passages (ragged,
                    padded), with shared key heads; for one new token, a few, or a prompt, with `rows` the ids that a search
                    found (-1: nothing found)
  RelativeBias      a learned position bias by buckets of the distance, added to the logits, and its gradient
  attend_backward   the gradients of queries, keys, values and of the bias table

A pass is one call as a user makes it: `attend` alone, or a training step's `attend` and `attend_backward`.
"""
import math

import torch

own = False

# The most work of a drawn case: bytes of states, logits of all heads (the plain form holds them in 32 bits), and flops.
MOST_STATE_BYTES, MOST_LOGITS, MOST_FLOPS = 3_400_000_000, 560_000_000, 980_000_000_000

BASE = {"batch": 1, "tokens": 1, "passages": 10, "length": 128, "heads": 8, "kv_heads": 8, "d": 64, "type": "bf16",
        "bank": 0, "ragged": False, "buckets": 0, "max_distance": 0, "two_sided": False, "later": False, "train": False}


def _case(name, **given):
    return {"name": name, **BASE, **given}


def listed():
    return [
        # One new token of one request over its ten found passages: the smallest call, latency alone counts.
        _case("token_1x10x64", passages=10, length=64, bank=1000),
        # A serving batch: one new token each over ten found passages of ragged lengths, shared key heads.
        _case("token_64x10x100", batch=64, passages=10, length=100, heads=16, kv_heads=4, d=128, type="f16", bank=2000,
              ragged=True),
        # One new token over a hundred found passages (the search's long result lists): the most states, bytes bound.
        _case("token_32x100x256", batch=32, passages=100, length=256, heads=32, kv_heads=8, d=128, bank=4000),
        # A few new tokens at each request's own position, with the reader's one-sided bias, of odd sizes.
        _case("tokens7_16x20x131", batch=16, tokens=7, passages=20, length=131, heads=12, kv_heads=6, d=96, bank=1001,
              ragged=True, buckets=32, max_distance=128, later=True),
        # A prompt over its found passages, each key head with its own query head.
        _case("prompt512_4x10x512", batch=4, tokens=512, passages=10, length=512, heads=16, kv_heads=16, bank=1000),
        # A long prompt over many passages: the largest forward, bound by the matrix products.
        _case("prompt4096_1x16x512", tokens=4096, passages=16, length=512, heads=16, kv_heads=4, d=128, bank=500),
        # Encoding a batch of queries for the search: short ragged texts with the two-sided bias, forward alone.
        _case("encode_256x128", batch=256, tokens=128, passages=1, length=128, heads=12, kv_heads=12, ragged=True,
              buckets=32, max_distance=128, two_sided=True),
        # A training step of the encoder that makes vectors and states: the two-sided bias and its gradient.
        _case("train_encoder_32x512", batch=32, tokens=512, passages=1, length=512, heads=12, kv_heads=12, buckets=32,
              max_distance=128, two_sided=True, train=True),
        # The same on long texts, where most of the logits share the two farthest buckets.
        _case("train_encoder_4x2048", batch=4, tokens=2048, passages=1, length=2048, heads=12, kv_heads=12, buckets=32,
              max_distance=128, two_sided=True, train=True),
        # A training step of a small reader: odd sizes everywhere, the one-sided bias, shared key heads.
        _case("train_reader_3x77_5x131", batch=3, tokens=77, passages=5, length=131, heads=6, kv_heads=3, d=80,
              type="f16", ragged=True, buckets=20, max_distance=100, train=True),
        # A training step of a reader over ragged passages, shared key heads.
        _case("train_reader_8x256_8x256", batch=8, tokens=256, passages=8, length=256, heads=16, kv_heads=8, d=128,
              ragged=True, train=True),
        # The largest training step: long targets over long passages.
        _case("train_reader_2x2048_4x2048", batch=2, tokens=2048, passages=4, length=2048, heads=16, kv_heads=16, d=128,
              train=True),
    ]


def _log_int(rng, lo, hi):
    """A whole number in [lo, hi], uniform over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    c = dict(BASE)
    kind = rng.choice(["token", "token", "tokens", "prompt", "encode", "train_encoder", "train_reader"])
    c["train"] = kind.startswith("train")
    c["type"] = rng.choice(["bf16", "bf16", "f16"])
    c["d"] = rng.choice([32, 40, 64, 64, 64, 80, 96, 128, 128, 128])
    c["kv_heads"] = rng.choice([1, 2, 4, 8, 12])
    c["heads"] = c["kv_heads"] * rng.choice([1, 1, 2, 4])
    c["ragged"] = rng.random() < 0.6
    itself = kind in ("encode", "train_encoder")
    if itself:
        c["passages"], c["length"] = 1, _log_int(rng, 16, 2048)
        c["tokens"] = c["length"]
    else:
        c["tokens"] = {"token": 1, "tokens": _log_int(rng, 2, 16)}.get(kind) or _log_int(rng, 17, 4096)
        c["passages"], c["length"] = _log_int(rng, 1, 16 if c["train"] else 100), _log_int(rng, 16, 512)
    if itself or rng.random() < 0.3:
        c["two_sided"] = itself
        c["buckets"], c["max_distance"] = rng.choice([(32, 128), (32, 128), (32, 256), (20, 100), (64, 512)])
        c["later"] = not itself and not c["train"]
    # the work decides what is left: passages first, then the batch
    one = lambda: {"bytes": c["passages"] * c["length"] * c["kv_heads"] * c["d"] * 4,
                   "logits": c["tokens"] * c["passages"] * c["length"] * c["heads"]}
    flops = lambda: one()["logits"] * c["d"] * (14 if c["train"] else 4)
    while one()["bytes"] > MOST_STATE_BYTES or one()["logits"] > MOST_LOGITS or flops() > MOST_FLOPS:
        c["passages" if c["passages"] > 1 else "tokens"] //= 2
    most = min(MOST_STATE_BYTES // one()["bytes"], MOST_LOGITS // one()["logits"], int(MOST_FLOPS // flops()), 256)
    c["batch"] = _log_int(rng, 1, max(1, most))
    if not itself and not c["train"]:  # a bank of states, from which the search found each query's rows
        c["bank"] = max(c["passages"], min(1000, int(MOST_STATE_BYTES // (one()["bytes"] // c["passages"]))))
    return c


def _dtype(case):
    return {"bf16": torch.bfloat16, "f16": torch.float16}[case["type"]]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    b, t, r, s = case["batch"], case["tokens"], case["passages"], case["length"]
    n = case["bank"] or b * r
    dtype = _dtype(case)

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g, dtype=dtype)

    state = {"case": case, "q": normal(b, t, case["heads"], case["d"]) * 1.5, "k": normal(n, s, case["kv_heads"], case["d"]),
             "v": normal(n, s, case["kv_heads"], case["d"]), "rows": None, "lengths": None, "table": None, "start": 0}
    if case["bank"]:
        # (dist, id) records as the search leaves them: distinct ids, and where it found less than it was asked for, -1
        found = torch.rand(b, n, device="cuda", generator=g).argsort(dim=1)[:, :r].to(torch.int32)
        kept = torch.randint(r - r // 8, r + 1, (b, 1), device="cuda", generator=g)
        found = torch.where(torch.arange(r, device="cuda") < kept, found, torch.full_like(found, -1))
        state["rows"] = torch.stack([torch.zeros_like(found), found], -1)[..., 1]
    if case["ragged"]:
        state["lengths"] = torch.randint(s // 4, s + 1, (n,), device="cuda", generator=g, dtype=torch.int32)
    if case["buckets"]:
        state["table"] = normal(case["buckets"], case["heads"])
    if case["later"]:  # where each request's new tokens stand
        state["start"] = torch.randint(0, 2 * s, (b,), device="cuda", generator=g, dtype=torch.int32)
    if case["train"]:
        state["d_out"] = normal(b, t, case["heads"], case["d"])
    return state


def _edges(side, max_distance):
    """The distances at which the buckets from side/2 + 1 on begin: the least x with
    (x/e)^(side-e) >= (max_distance/e)^i, e = side/2, in whole numbers."""
    e = side // 2
    w = side - e
    found, x = [], e
    for i in range(1, w):
        while x ** w * e ** i < max_distance ** i * e ** w:
            x += 1
        found.append(x)
    return found


def _bucket(case, x):
    """The bucket of each distance x = key position - query position."""
    side = case["buckets"] // 2 if case["two_sided"] else case["buckets"]
    e = side // 2
    a = x.abs() if case["two_sided"] else (-x).clamp(min=0)
    edges = torch.tensor(_edges(side, case["max_distance"]), device=x.device)
    far = e + torch.bucketize(a, edges, right=True)
    return torch.where(a < e, a, far) + (side * (x > 0) if case["two_sided"] else 0)


def _plain(state):
    """The operators from elementary operations in 32 bits, with all logits held at once."""
    case = state["case"]
    b, t, r, s, h, hk, d = (case[x] for x in ("batch", "tokens", "passages", "length", "heads", "kv_heads", "d"))
    share, n, dtype = h // hk, state["k"].shape[0], state["q"].dtype
    rows = state["rows"] if state["rows"] is not None else torch.arange(b * r, device="cuda").view(b, r)
    at = rows.clamp(min=0).long()
    lengths = state["lengths"] if state["lengths"] is not None else torch.full((n,), s, device="cuda")
    there = (torch.arange(s, device="cuda") < lengths[at][..., None]) & (rows >= 0)[..., None]  # [b, r, s]
    there = there.view(b, 1, 1, r * s)

    def heads_first(x):  # [b, keys, hk, d] -> [b, hk, keys, d]
        return x.float().transpose(1, 2).contiguous()

    def grouped(x):  # [b, t, h, d] -> [b, hk, share * t, d]
        return x.float().view(b, t, hk, share, d).permute(0, 2, 3, 1, 4).reshape(b, hk, share * t, d)

    def ungrouped(x):
        return x.view(b, hk, share, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, h, d)

    q = grouped(state["q"])
    if state["rows"] is None:
        k, v = heads_first(state["k"].view(b, r * s, hk, d)), heads_first(state["v"].view(b, r * s, hk, d))
    else:
        k, v = heads_first(state["k"][at].view(b, r * s, hk, d)), heads_first(state["v"][at].view(b, r * s, hk, d))
    scale = 1 / math.sqrt(d)
    logits = (torch.matmul(q, k.transpose(2, 3).contiguous()) * scale).view(b, hk, share, t, r * s)
    bucket = None
    if case["buckets"]:
        start = state["start"].view(b, 1, 1) if case["later"] else torch.zeros(1, 1, 1, device="cuda", dtype=torch.int32)
        x = torch.arange(s, device="cuda").repeat(r) - (torch.arange(t, device="cuda")[:, None] + start)
        bucket = _bucket(case, x)  # [b or 1, t, keys]
        bias = state["table"].float()[bucket]  # [b or 1, t, keys, h]
        logits += bias.permute(0, 3, 1, 2).reshape(bucket.shape[0], hk, share, t, r * s)
        del bias
    logits = logits.masked_fill_(~there[:, :, None], -math.inf)
    top = logits.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = logits.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, torch.ones_like(total), total)).view(b, hk, share * t, r * s)
    out = torch.matmul(p, v)
    if not case["train"]:
        return ungrouped(out).to(dtype)
    d_out = grouped(state["d_out"])
    d_p = torch.matmul(d_out, v.transpose(2, 3).contiguous())
    d_v = torch.matmul(p.transpose(2, 3).contiguous(), d_out)
    d_s = d_p.sub_((d_out * out).sum(-1, keepdim=True)).mul_(p)
    d_q = torch.matmul(d_s, k) * scale
    d_k = torch.matmul(d_s.transpose(2, 3).contiguous(), q) * scale
    found = {"out": ungrouped(out).to(dtype), "q": ungrouped(d_q).to(dtype)}
    found["k"] = d_k.transpose(1, 2).reshape(b * r, s, hk, d).to(dtype)
    found["v"] = d_v.transpose(1, 2).reshape(b * r, s, hk, d).to(dtype)
    if case["buckets"]:
        per_place = d_s.view(b, h, t, r * s).sum(0).reshape(h, t * r * s)
        chosen = (bucket[0].reshape(-1, 1) == torch.arange(case["buckets"], device="cuda")).float()
        found["table"] = torch.matmul(per_place, chosen).t().contiguous().to(dtype)
    return found


def run(state):
    if not own:
        return _plain(state)
    from veckern_amd import attention

    case = state["case"]
    bias = None
    if case["buckets"]:
        bias = attention.RelativeBias(state["table"], max_distance=case["max_distance"], two_sided=case["two_sided"])
    if not case["train"]:
        return attention.attend(state["q"], state["k"], state["v"], rows=state["rows"], lengths=state["lengths"], bias=bias,
                                q_start=state["start"])
    out, lse = attention.attend(state["q"], state["k"], state["v"], lengths=state["lengths"], bias=bias,
                                q_start=state["start"], return_lse=True)
    grad = attention.attend_backward(state["d_out"], state["q"], state["k"], state["v"], out, lse,
                                     lengths=state["lengths"], bias=bias, q_start=state["start"])
    found = {"out": out, "q": grad.queries, "k": grad.keys, "v": grad.values}
    if bias is not None:
        found["table"] = grad.table
    return found


def work(case):
    b, t, r, s, h, hk, d = (case[x] for x in ("batch", "tokens", "passages", "length", "heads", "kv_heads", "d"))
    filled = 0.625 if case["ragged"] else 1.0  # the mean of lengths that are uniform from a quarter to the whole
    read = float(b * r)  # rows that are attended to, and how many of them are distinct
    distinct = read
    if case["bank"]:
        read = b * (r - (r // 8) / 2)
        distinct = case["bank"] * (1 - (1 - 1 / case["bank"]) ** read)
    one_q, one_k = b * t * h * d * 2, distinct * s * filled * hk * d * 2
    pairs = t * h * read * s * filled
    if not case["train"]:
        return {"bytes": 2 * one_q + 2 * one_k, "flops": 4 * pairs * d}
    # q, k, v and d_out come in once, out and the three gradients leave once (gradients of absent states are zeros)
    return {"bytes": 4 * one_q + 2 * one_k + 2 * b * r * s * hk * d * 2, "flops": 14 * pairs * d}


def exact(case, seed):
    """The definition in 64 bits, one request and key head at a time, each key there gathered first."""
    b, t, r, s, h, hk, d = (case[x] for x in ("batch", "tokens", "passages", "length", "heads", "kv_heads", "d"))
    state = prepare(case, seed)
    share = h // hk
    dev = state["q"].device
    n = state["k"].shape[0]
    rows = (torch.arange(b * r).view(b, r) if state["rows"] is None else state["rows"]).tolist()
    lengths = [s] * n if state["lengths"] is None else state["lengths"].tolist()
    start = state["start"].tolist() if case["later"] else [0] * b
    out = torch.zeros(b, t, h, d, dtype=torch.float64, device=dev)
    dq, table = torch.zeros_like(out), torch.zeros(h, max(1, case["buckets"]), dtype=torch.float64, device=dev)
    dk = torch.zeros(n if case["train"] else 0, s, hk, d, dtype=torch.float64, device=dev)
    dv = torch.zeros_like(dk)
    side = case["buckets"] // 2 if case["two_sided"] else case["buckets"]
    for i in range(b):
        held = [(n_, x) for n_ in rows[i] if n_ >= 0 for x in range(lengths[n_])]
        if not held:
            continue
        row, pos = torch.tensor(held, device=dev).t()
        gap = pos[None, :] - (torch.arange(t, device=dev)[:, None] + start[i])
        if case["buckets"]:
            e = side // 2
            a = (gap.abs() if case["two_sided"] else (-gap).clamp(min=0)).double()
            far = e + torch.floor(torch.log(a.clamp(min=e) / e) / math.log(case["max_distance"] / e) * (side - e) + 1e-9)
            place = torch.where(a < e, a, far.clamp(max=side - 1)).long()
            if case["two_sided"]:
                place = place + side * (gap > 0)
        for j in range(hk):
            k, v = state["k"][row, pos, j].double(), state["v"][row, pos, j].double()
            for m in range(j * share, (j + 1) * share):
                q = state["q"][i, :, m].double()
                logit = q @ k.t().contiguous() / math.sqrt(d)
                if case["buckets"]:
                    logit = logit + state["table"][:, m].double()[place]
                p = torch.exp(logit - torch.logsumexp(logit, -1, keepdim=True))
                out[i, :, m] = p @ v
                if case["train"]:
                    do = state["d_out"][i, :, m].double()
                    ds = do @ v.t().contiguous()
                    ds = p * (ds - (p * ds).sum(-1, keepdim=True))
                    dq[i, :, m] = ds @ k / math.sqrt(d)
                    dk[row, pos, j] += ds.t().contiguous() @ q / math.sqrt(d)
                    dv[row, pos, j] += p.t().contiguous() @ do
                    if case["buckets"]:
                        table[m] += torch.bincount(place.reshape(-1), weights=ds.reshape(-1), minlength=case["buckets"])
    if not case["train"]:
        return out
    found = {"out": out, "q": dq, "k": dk, "v": dv}
    if case["buckets"]:
        found["table"] = table.t().contiguous()
    return found
