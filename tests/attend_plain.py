"""The attention over found rows and its gradients in 64 bits on the CPU, from the formulas, with the error that a kernel's
declared roundings can make in each result (u: unit roundoff of the type: 2^-8 for
bfloat16 with its 8 significant bits, 2^-11 for binary16 with its 11).

The kernels multiply inputs exactly into 32-bit sums, round P and dS to the type where they are multiplied again, and round
each result once. So, with FP32 = 1e-5 as the allowance for 32-bit logits, exponentials and sums (logits here stay below 50
and head sizes below 129: 50 * 2^-24 + 128 * 2^-24 stays below it), element by element:
  out    u sum P|v| + u|out|                      (+ 2^-25 sum |v| where P can be subnormal in binary16)
  delta  sum |dO| err(out)
  dv     u sum P|dO| + u|dv|
  dq     scale sum (u|dS| + P err(delta)) |k| + u|dq|,   dk alike
  table  sum P err(delta) + u|table|
each plus FP32 times the sum of the absolute values that were added."""
import math

import torch

FP32 = 1e-5


def unit(dtype):
    return {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float64: 0.0}[dtype]


def least(dtype):
    """Half the spacing of the type's subnormal numbers, for results that are so small."""
    return {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float64: 0.0}[dtype]


def bucket(x, buckets, max_distance, two_sided):
    """The bucket of one distance, in whole numbers: (a / e)^(n - e) against (max_distance / e)^i."""
    n = buckets // 2 if two_sided else buckets
    e = n // 2
    a = abs(x) if two_sided else max(-x, 0)
    found = a
    if a >= e:
        i = 0
        while i < n - e - 1 and a ** (n - e) * e ** (i + 1) >= max_distance ** (i + 1) * e ** (n - e):
            i += 1
        found = e + i
    return found + (n if two_sided and x > 0 else 0)


def plain(q, k, v, *, rows=None, lengths=None, table=None, buckets=0, max_distance=0, two_sided=False, q_start=0,
          scale=None, d_out=None):
    """Every result and its allowed error: {"out": (value, error), "lse": ..., and with d_out "q", "k", "v", "table"}."""
    u, tiny = unit(q.dtype), least(q.dtype)
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    batch, tokens, heads, d = q.shape
    bank, length, kv_heads, _ = k.shape
    share = heads // kv_heads
    passages = (bank // batch if batch else 0) if rows is None else rows.shape[1]
    rows = torch.arange(batch * passages).view(batch, passages) if rows is None else rows.cpu()
    lengths = torch.full((bank,), length) if lengths is None else lengths.cpu().clamp(0, length)
    start = q_start.cpu().tolist() if isinstance(q_start, torch.Tensor) else [q_start] * batch
    scale = 1 / math.sqrt(d) if scale is None else scale
    table = None if table is None else table.detach().cpu().double()
    got = {"out": (torch.zeros(batch, tokens, heads, d).double(), torch.zeros(batch, tokens, heads, d).double()),
           "lse": (torch.full((batch, heads, tokens), -math.inf).double(), torch.zeros(batch, heads, tokens).double())}
    if d_out is not None:
        d_out = d_out.detach().cpu().double()
        for name, like in (("q", q), ("k", k), ("v", v)) + ((("table", table),) if table is not None else ()):
            got[name] = (torch.zeros(like.shape).double(), torch.zeros(like.shape).double())
    for b in range(batch):
        held = [(n, s) for n in rows[b].tolist() if 0 <= n < bank for s in range(int(lengths[n]))]
        if not held:
            continue
        row, pos = torch.tensor(held).t()
        place = None
        if table is not None:
            place = torch.tensor([[bucket(s - t - start[b], buckets, max_distance, two_sided) for s in pos.tolist()]
                                  for t in range(tokens)], dtype=torch.long).view(tokens, len(held))
        for h in range(heads):
            kk, vv, qq = k[row, pos, h // share], v[row, pos, h // share], q[b, :, h]
            logit = qq @ kk.t() * scale
            if table is not None:
                logit = logit + table[:, h][place]
            top = logit.amax(-1, keepdim=True)
            full = (top != -math.inf).squeeze(-1)
            p = torch.where(full[:, None], torch.exp(logit - torch.where(full[:, None], top, 0.0)), 0.0)
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(full[:, None], total, 1.0)
            o = p @ vv
            o_err = (u + FP32) * (p @ vv.abs()) + u * o.abs() + 2 * tiny * (vv.abs().sum(0) * full[:, None] + 1)
            got["out"][0][b, :, h], got["out"][1][b, :, h] = o, o_err
            got["lse"][0][b, h] = torch.where(full, top.squeeze(-1) + torch.log(total.squeeze(-1)), -math.inf)
            got["lse"][1][b, h] = FP32 * (1 + logit.abs().clamp(max=1e30).amax(-1))
            if d_out is None:
                continue
            do = d_out[b, :, h]
            dp = do @ vv.t()
            delta = (p * dp).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            delta_err = (do.abs() * (o_err + FP32 * o.abs())).sum(-1, keepdim=True)
            fp32 = FP32 * p * (do.abs() @ vv.abs().t() + delta.abs())
            ds_err = p * delta_err + fp32 + u * ds.abs() + tiny
            for name, value, error in (("q", ds @ kk * scale, ds_err @ kk.abs() * scale),):
                got[name][0][b, :, h] = value
                got[name][1][b, :, h] = error + u * value.abs() + tiny
            got["k"][0][row, pos, h // share] += ds.t() @ qq * scale
            got["k"][1][row, pos, h // share] += ds_err.t() @ qq.abs() * scale
            got["v"][0][row, pos, h // share] += p.t() @ do
            got["v"][1][row, pos, h // share] += ((u + FP32) * p + tiny).t() @ do.abs()
            if table is not None:
                for c in range(buckets):
                    here = place == c
                    got["table"][0][c, h] += (ds * here).sum()
                    got["table"][1][c, h] += ((p * delta_err + fp32) * here).sum()
    for name in ("k", "v", "table"):
        if name in got:
            got[name] = (got[name][0], got[name][1] + u * got[name][0].abs() + tiny)
    return got


def check(name, result, got):
    """`result` within the allowed error of got[name]; infinite values equal."""
    value, error = got[name]
    x = result.detach().cpu().double()
    assert x.shape == value.shape, (name, x.shape, value.shape)
    fine = torch.isfinite(value)
    assert torch.equal(x[~fine], value[~fine]), f"{name}: infinite values differ"
    assert torch.isfinite(x[fine]).all(), f"{name}: not finite"
    off = (x - value).abs()[fine]
    over = off > error[fine]
    assert not over.any(), f"{name}: {int(over.sum())} of {over.numel()} off, by up to {float((off / error[fine].clamp(min=1e-300)).max()):.3g} times the allowed error"
