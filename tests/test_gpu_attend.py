"""Attention over found rows (veckern_amd.attention): forward, position bias, gradients, against 64 bits on the CPU."""
import math

import pytest

torch = pytest.importorskip("torch")

import veckern_amd as vk
from tests.attend_plain import check, plain

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def make(seed, dtype, batch, tokens, passages, length, heads, kv_heads, d, bank=0, ragged=False, empty=()):
    g = torch.Generator().manual_seed(seed)
    n = bank or batch * passages

    def normal(*shape):
        return torch.randn(*shape, generator=g).to(dtype).cuda()

    rows = None
    if bank:
        rows = torch.randint(0, bank, (batch, passages), generator=g, dtype=torch.int32).cuda()
    lengths = None
    if ragged:
        lengths = torch.randint(0, length + 1, (n,), generator=g, dtype=torch.int32)
        for i in empty:
            lengths[i] = 0
        lengths = lengths.cuda()
    return (normal(batch, tokens, heads, d) * 1.5, normal(n, length, kv_heads, d), normal(n, length, kv_heads, d),
            rows, lengths, normal(batch, tokens, heads, d))


def both(q, k, v, rows=None, lengths=None, table=None, buckets=0, max_distance=128, two_sided=True, q_start=0, scale=None,
         d_out=None, got=None):
    """Runs the kernels, checks every result against plain(), and returns them."""
    from veckern_amd import attention

    bias = None if table is None else attention.RelativeBias(table, max_distance, two_sided)
    if got is None:
        got = plain(q, k, v, rows=rows, lengths=lengths, table=table, buckets=buckets, max_distance=max_distance,
                    two_sided=two_sided, q_start=q_start, scale=scale, d_out=d_out)
    out, lse = attention.attend(q, k, v, rows=rows, lengths=lengths, bias=bias, q_start=q_start, scale=scale, return_lse=True)
    check("out", out, got)
    check("lse", lse.double().sum(-1), got)
    if d_out is None:
        return out, lse
    grad = attention.attend_backward(d_out, q, k, v, out, lse, rows=rows, lengths=lengths, bias=bias, q_start=q_start,
                                     scale=scale)
    check("q", grad.queries, got)
    if rows is None:
        check("k", grad.keys, got)
        check("v", grad.values, got)
    else:
        assert grad.keys is None and grad.values is None
    if table is not None:
        check("table", grad.table, got)
    return out, lse, grad


# tokens from one to past a block's columns, passages that end inside a tile and fill it, one position, shared heads
SHAPES = [
    # batch, tokens, passages, length, heads, kv_heads, d, bank, ragged
    (1, 1, 1, 1, 1, 1, 8, 0, False),
    (1, 1, 10, 64, 8, 8, 64, 50, False),
    (3, 1, 7, 100, 16, 4, 128, 40, True),
    (2, 1, 3, 33, 6, 1, 72, 9, True),
    (5, 7, 4, 131, 12, 6, 96, 30, True),
    (2, 16, 2, 65, 4, 2, 64, 9, True),
    (1, 33, 5, 63, 2, 2, 40, 0, True),
    (2, 77, 5, 130, 6, 3, 80, 0, True),
    (2, 128, 1, 128, 4, 4, 64, 0, False),
    (1, 129, 1, 257, 4, 1, 128, 0, False),
    (1, 300, 3, 70, 2, 1, 16, 0, True),
    # many short passages: several in a tile, more than a block holds the rows of
    (2, 40, 9, 17, 4, 2, 64, 0, True),
    (3, 45, 30, 7, 2, 2, 128, 0, True),
    (1, 3, 300, 5, 2, 1, 64, 40, True),
    (1, 70, 600, 3, 2, 2, 128, 50, True),
    (2, 1, 70, 33, 4, 1, 72, 40, True),
    (1, 50, 280, 20, 1, 1, 32, 0, False),
]


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_gradients(shape, dtype):
    batch, tokens, passages, length, heads, kv_heads, d, bank, ragged = shape
    q, k, v, rows, lengths, d_out = make(11, dtype, batch, tokens, passages, length, heads, kv_heads, d, bank, ragged)
    both(q, k, v, rows, lengths, d_out=d_out)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("kind", [(32, 128, True), (32, 128, False), (20, 100, False), (6, 9, True), (2, 2, False), (64, 512, True),
                                  (7, 40, False)], ids=str)
@pytest.mark.parametrize("shape", [(2, 150, 1, 150, 3, 3, 64, 0, True), (2, 70, 2, 200, 4, 2, 80, 0, False),
                                   (3, 5, 4, 131, 6, 2, 128, 11, True), (1, 1, 3, 40, 4, 4, 64, 5, False),
                                   (2, 60, 11, 21, 2, 1, 64, 0, True), (1, 33, 7, 50, 2, 2, 128, 0, True),
                                   (1, 90, 5, 37, 2, 2, 64, 9, True)], ids=str)
def test_position_bias(shape, kind, dtype):
    batch, tokens, passages, length, heads, kv_heads, d, bank, ragged = shape
    buckets, max_distance, two_sided = kind
    q, k, v, rows, lengths, d_out = make(12, dtype, batch, tokens, passages, length, heads, kv_heads, d, bank, ragged)
    g = torch.Generator().manual_seed(5)
    table = torch.randn(buckets, heads, generator=g).to(dtype).cuda()
    start = torch.randint(-30, 2 * length, (batch,), generator=g, dtype=torch.int32).cuda() if bank else 0
    both(q, k, v, rows, lengths, table, buckets, max_distance, two_sided, start, d_out=d_out)


@pytest.mark.parametrize("two_sided", [True, False])
@pytest.mark.parametrize("d", [32, 64, 80, 128])
def test_wide_position_bias_over_many_blocks(d, two_sided):
    """More blocks than compute units, and buckets so wide that the table's gradient is summed without a tile in LDS."""
    batch, tokens, heads = 34, 9, 8
    q, k, v, _, lengths, d_out = make(d, BF16, batch, tokens, 3, 70, heads, 4, d, 0, True)
    table = torch.randn(64, heads, generator=torch.Generator().manual_seed(d)).to(BF16).cuda()
    both(q, k, v, lengths=lengths, table=table, buckets=64, max_distance=512, two_sided=two_sided, q_start=35, d_out=d_out)


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("shape", [(1, 900, 2, 40, 8, 2, 64, 0, True), (1, 1100, 1, 50, 4, 4, 24, 0, False),
                                   (1, 700, 3, 33, 8, 2, 128, 0, True), (2, 515, 1, 19, 6, 2, 96, 0, False)], ids=str)
def test_many_tokens_over_few_states(shape, biased):
    """The states' gradient is summed over query tiles by several blocks."""
    q, k, v, _, lengths, d_out = make(31, BF16, *shape)
    bias = {}
    if biased:
        table = torch.randn(32, shape[4], generator=torch.Generator().manual_seed(32)).to(BF16).cuda()
        bias = dict(table=table, buckets=32, max_distance=128, two_sided=True)
    both(q, k, v, lengths=lengths, d_out=d_out, **bias)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("length", [15, 40])
def test_many_ragged_passages(d, length):
    """Slots that hold a key are found over more passages than a wave has lanes, most of them empty in one request."""
    batch, passages = 2, 150
    q, k, v, _, lengths, d_out = make(d + length, BF16, batch, 20, passages, length, 4, 2, d, 0, True, empty=range(0, 130))
    table = torch.randn(16, 4, generator=torch.Generator().manual_seed(d)).to(BF16).cuda()
    both(q, k, v, lengths=lengths, d_out=d_out, table=table, buckets=16, max_distance=20, two_sided=True)


@pytest.mark.parametrize("shape", [(2, 150, 5, 23, 4, 2, 32, 12, True), (3, 40, 9, 7, 2, 2, 16, 0, True),
                                   (1, 300, 1, 190, 2, 1, 24, 0, False)], ids=str)
def test_small_heads(shape):
    q, k, v, rows, lengths, d_out = make(41, F16, *shape)
    both(q, k, v, rows=rows, lengths=lengths, d_out=d_out)


@pytest.mark.parametrize("start", [-700, -1, 3, 90, 5000])
def test_position_of_the_first_token(start):
    q, k, v, _, _, d_out = make(13, BF16, 1, 66, 2, 100, 2, 2, 64)
    table = torch.randn(32, 2, generator=torch.Generator().manual_seed(6)).to(BF16).cuda()
    both(q, k, v, table=table, buckets=32, max_distance=128, two_sided=True, q_start=start, d_out=d_out)


def test_long_rows_and_many_splits():
    q, k, v, rows, lengths, _ = make(14, BF16, 2, 3, 9, 1500, 4, 2, 64, 20, True)
    both(q, k, v, rows, lengths)
    q, k, v, rows, lengths, d_out = make(15, F16, 1, 20, 2, 3000, 2, 1, 128)
    both(q, k, v, rows, lengths, d_out=d_out)


def test_rows_that_are_not_there():
    q, k, v, rows, lengths, d_out = make(16, BF16, 4, 5, 6, 50, 4, 2, 64, 12, True, empty=(3, 4))
    rows[0] = -1                                                           # nothing found
    rows[1] = torch.tensor([12, -1, 2**31 - 1, -2**31, 3, 4])              # outside the bank, or of length zero
    rows[2] = 7                                                            # the same row six times
    lengths[7] = 13
    lengths[8] = 10_000                                                    # more than there is: all of it
    lengths[9] = -5
    rows[3, :2] = torch.tensor([8, 9])
    out, lse, grad = both(q, k, v, rows, lengths, d_out=d_out)
    for b in (0, 1):
        assert (out[b] == 0).all() and (lse[b, ..., 0] == -math.inf).all() and (grad.queries[b] == 0).all()


def test_records_of_a_search_are_read_where_they_lie():
    q, k, v, rows, lengths, _ = make(17, F16, 3, 1, 10, 64, 4, 4, 64, 40, True)
    records = torch.stack([torch.full_like(rows, 123456), rows], -1)[..., 1]
    assert records.stride() == (20, 2)
    from veckern_amd import attention

    assert torch.equal(attention.attend(q, k, v, rows=records, lengths=lengths),
                       attention.attend(q, k, v, rows=rows, lengths=lengths))


@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_what_lies_in_absent_places_does_not_matter(poison):
    from veckern_amd import attention

    q, k, v, rows, lengths, d_out = make(18, BF16, 2, 40, 3, 100, 4, 2, 64, 0, True, empty=(1,))
    table = torch.randn(32, 4, generator=torch.Generator().manual_seed(7)).to(BF16).cuda()
    bias = attention.RelativeBias(table)

    def all_of(k, v):
        out, lse = attention.attend(q, k, v, lengths=lengths, bias=bias, return_lse=True)
        return (out, lse, *attention.attend_backward(d_out, q, k, v, out, lse, lengths=lengths, bias=bias))

    clean = all_of(k, v)
    absent = torch.arange(100, device="cuda")[None] >= lengths[:, None]
    k[absent], v[absent] = poison, poison
    for x, y in zip(clean, all_of(k, v)):
        assert torch.equal(x, y)
    for x in clean[3:5]:
        assert (x[absent] == 0).all()


def test_bias_of_minus_infinity_and_of_the_lowest_value():
    q, k, v, _, _, d_out = make(19, BF16, 1, 40, 1, 90, 2, 2, 64)
    table = torch.randn(32, 2, generator=torch.Generator().manual_seed(8)).to(BF16)
    table[3:, 0] = -math.inf                      # one-sided: head 0 sees the keys up to two before the query, and those after
    table[:, 1] = torch.finfo(BF16).min           # head 1: equal and lowest everywhere: as if no logit mattered
    both(q, k, v, table=table.cuda(), buckets=32, max_distance=128, two_sided=False, d_out=d_out)
    table[:, 0] = -math.inf                       # nothing is left for head 0
    out, lse, grad = both(q, k, v, table=table.cuda(), buckets=32, max_distance=128, two_sided=False, d_out=d_out)
    assert (out[:, :, 0] == 0).all() and (lse[:, 0, :, 0] == -math.inf).all() and (grad.queries[:, :, 0] == 0).all()


def test_large_logits_and_scale():
    q, k, v, _, _, d_out = make(20, BF16, 1, 50, 1, 120, 2, 2, 64)
    both(q, k, v, scale=0.6, d_out=d_out)         # logits to about 40: weights from 1 to 0
    both(q, k, v, scale=0.0, d_out=d_out)         # all weights equal


@pytest.mark.parametrize("sizes", [(0, 4, 0, 8), (2, 0, 3, 8), (2, 4, 0, 8), (2, 4, 3, 0)], ids=str)
def test_nothing_to_do(sizes):
    batch, tokens, passages, length = sizes
    for with_rows in (False, True):
        q = torch.ones(batch, tokens, 4, 16, dtype=F16, device="cuda")
        k = torch.ones(batch * passages, length, 2, 16, dtype=F16, device="cuda")
        rows = torch.zeros(batch, passages, dtype=torch.int32, device="cuda") if with_rows else None
        table = torch.ones(8, 4, dtype=F16, device="cuda")
        both(q, k, k.clone(), rows, None, table, 8, 20, True, d_out=q.clone())


def test_layouts_that_are_not_contiguous():
    g = torch.Generator().manual_seed(21)
    batch, tokens, heads, d = 2, 70, 4, 64
    fused = torch.randn(batch, tokens, 3, heads, d, generator=g).to(BF16).cuda()      # one projection's output
    q, k, v = fused.unbind(2)
    d_out = torch.randn(batch, heads, tokens, d, generator=g).to(BF16).cuda().transpose(1, 2)
    both(q, k, v, d_out=d_out)
    heads_first = torch.randn(2, heads, tokens, d, generator=g).to(BF16).cuda().transpose(1, 2)
    both(heads_first, heads_first, v, d_out=d_out)
    one = torch.randn(1, 90, 2, d, generator=g).to(BF16).cuda()                        # one row's states for both requests
    both(q, one.expand(2, 90, 2, d), one.expand(2, 90, 2, d), d_out=d_out)
    table = torch.randn(heads, 32, generator=g).to(BF16).cuda().t()
    from veckern_amd import attention

    x = attention.attend(q, k, v, bias=attention.RelativeBias(table))
    assert torch.equal(x, attention.attend(q, k, v, bias=attention.RelativeBias(table.contiguous())))


def test_gradients_against_differences():
    """The derivative along a direction, by differences of the 64-bit loss, against the kernels' gradients."""
    from veckern_amd import attention

    q, k, v, _, lengths, d_out = make(22, BF16, 2, 20, 3, 40, 4, 2, 32, 0, True)
    table = torch.randn(12, 4, generator=torch.Generator().manual_seed(9)).to(BF16).cuda()
    kind = dict(buckets=12, max_distance=30, two_sided=True)
    got = plain(q, k, v, lengths=lengths, table=table, d_out=d_out, **kind)
    bias = attention.RelativeBias(table, 30, True)
    out, lse = attention.attend(q, k, v, lengths=lengths, bias=bias, return_lse=True)
    grad = attention.attend_backward(d_out, q, k, v, out, lse, lengths=lengths, bias=bias)
    g = torch.Generator().manual_seed(10)
    inputs = {"q": q, "k": k, "v": v, "table": table}
    results = {"q": grad.queries, "k": grad.keys, "v": grad.values, "table": grad.table}

    def loss(moved):
        full = {n: x.detach().cpu().double() for n, x in inputs.items()}
        full.update(moved)
        o = plain(full["q"], full["k"], full["v"], lengths=lengths, table=full["table"], **kind)["out"][0]
        return float((o * d_out.cpu().double()).sum())

    for name, x in inputs.items():
        way = torch.randn(x.shape, generator=g).double()
        h = 1e-4
        at = x.cpu().double()
        slope = (loss({name: at + h * way}) - loss({name: at - h * way})) / (2 * h)
        ours = float((results[name].cpu().double() * way).sum())
        allowed = float((got[name][1] * way.abs()).sum()) + 1e-6 * abs(slope) + 1e-6
        assert abs(slope - ours) <= allowed, (name, slope, ours, allowed)


@pytest.mark.parametrize("d", [32, 64, 128])
def test_gradients_of_rows_with_one_key(d):
    """A softmax over one key is constant: no gradient reaches queries, keys or table, whatever the output was rounded to."""
    from veckern_amd import attention

    q, k, v, _, _, d_out = make(51, BF16, 3, 40, 1, 30, 4, 2, d)
    lengths = torch.ones(3, dtype=torch.int32, device="cuda")
    table = torch.randn(8, 4, generator=torch.Generator().manual_seed(52)).to(BF16).cuda()
    bias = attention.RelativeBias(table, 10, True)
    out, lse = attention.attend(q, k, v, lengths=lengths, bias=bias, return_lse=True)
    grad = attention.attend_backward(d_out, q, k, v, out, lse, lengths=lengths, bias=bias)
    # dP and the sum of P dP differ by what 32 bits leave: P is 1 up to 2^-18 (an exponent of at most 2^4, in steps of 2^-20,
    # and the exponential's own error), so that |dS| <= 2^-17 |dP|
    dp = (d_out.double().abs() * v[:, :1].double().abs().repeat_interleave(2, dim=2)).sum(-1)
    most = float(dp.max()) * 2.0 ** -17
    assert float(grad.queries.abs().max()) <= most * float(k.abs().max()) / d ** 0.5
    assert float(grad.keys.abs().max()) <= most * 40 * 2 * float(q.abs().max()) / d ** 0.5
    assert float(grad.table.abs().max()) <= most * 3 * 40


def test_automatic_differentiation():
    from veckern_amd import attention

    q, k, v, _, lengths, d_out = make(23, BF16, 2, 30, 2, 50, 4, 2, 64, 0, True)
    table = torch.randn(32, 4, generator=torch.Generator().manual_seed(11)).to(BF16).cuda()
    leaves = [x.clone().requires_grad_() for x in (q, k, v, table)]
    out = attention.attend(*leaves[:3], lengths=lengths, bias=attention.RelativeBias(leaves[3]))
    out.backward(d_out)
    _, _, grad = both(q, k, v, lengths=lengths, table=table, buckets=32, d_out=d_out)
    for x, y in zip(leaves, grad):
        assert torch.equal(x.grad, y)
    # a sum's gradient is one repeated element
    leaves[0].grad = None
    attention.attend(leaves[0], k, v, lengths=lengths).sum().backward()
    assert torch.isfinite(leaves[0].grad).all()
    # queries over a bank by rows have a gradient, the bank has none
    rows = torch.tensor([[1, 0], [3, -1]], dtype=torch.int32, device="cuda")
    leaves[0].grad = None
    attention.attend(leaves[0], k, v, rows=rows).backward(d_out)
    assert leaves[0].grad.abs().sum() > 0
    with pytest.raises(vk.VkInvalidArgument):
        attention.attend(leaves[0], leaves[1], v, rows=rows)


def test_same_bits_every_time_and_on_another_stream():
    from veckern_amd import attention

    q, k, v, _, lengths, d_out = make(24, BF16, 3, 200, 2, 300, 4, 2, 64, 0, True)
    bias = attention.RelativeBias(torch.randn(32, 4, generator=torch.Generator().manual_seed(12)).to(BF16).cuda())

    def all_of():
        out, lse = attention.attend(q, k, v, lengths=lengths, bias=bias, return_lse=True)
        return (out, lse, *attention.attend_backward(d_out, q, k, v, out, lse, lengths=lengths, bias=bias))

    first = all_of()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = all_of()
    torch.cuda.current_stream().wait_stream(stream)
    for x, y, z in zip(first, second, all_of()):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_captured_in_a_graph():
    from veckern_amd import attention

    q, k, v, rows, lengths, _ = make(25, F16, 4, 1, 10, 200, 8, 2, 128, 60, True)
    eager = attention.attend(q, k, v, rows=rows, lengths=lengths)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        attention.attend(q, k, v, rows=rows, lengths=lengths)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attention.attend(q, k, v, rows=rows, lengths=lengths)
    for i in range(4):
        out.zero_()
        q.copy_(q.roll(1, 0))
        eager = attention.attend(q, k, v, rows=rows, lengths=lengths)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager), i


def test_refusals():
    from veckern_amd import attention

    q, k, v, rows, lengths, _ = make(26, BF16, 2, 3, 2, 20, 4, 2, 64, 9, True)
    table = torch.zeros(32, 4, dtype=BF16, device="cuda")

    def refused(*args, **kw):
        with pytest.raises(vk.VkInvalidArgument):
            attention.attend(*args, **kw)

    refused(q.float(), k.float(), v.float(), rows=rows)
    refused(q, k.to(F16), v.to(F16), rows=rows)
    refused(q.cpu(), k, v, rows=rows)
    refused(q, k, v)                                             # 9 rows for 2 requests
    refused(q, k, v[:, :19], rows=rows)
    refused(q[..., :60], k[..., :60], v[..., :60], rows=rows)    # not a multiple of 8
    refused(q[..., 4:12], k[..., 4:12], v[..., 4:12], rows=rows)  # not aligned
    refused(q[:, :, :3], k, v, rows=rows)                        # 3 query heads over 2
    refused(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, rows=rows)
    refused(torch.zeros(2, 3, 4, 136, dtype=BF16, device="cuda"), *[torch.zeros(9, 20, 2, 136, dtype=BF16, device="cuda")] * 2,
            rows=rows)
    refused(q, k, v, rows=rows.long())
    refused(q, k, v, rows=rows[:1])
    refused(q, k, v, rows=rows, lengths=lengths[:8])
    refused(q, k, v, rows=rows, lengths=lengths.long())
    refused(q, k, v, rows=rows, scale=math.nan)
    refused(q, k, v, rows=rows, scale=-1.0)
    refused(q, k, v, rows=rows, bias=attention.RelativeBias(table[:, :3]))
    refused(q, k, v, rows=rows, bias=attention.RelativeBias(table.to(F16)))
    refused(q, k, v, rows=rows, bias=attention.RelativeBias(table[:31]))                     # odd, two-sided
    refused(q, k, v, rows=rows, bias=attention.RelativeBias(table[:1], two_sided=False))
    refused(q, k, v, rows=rows, bias=attention.RelativeBias(table, max_distance=8))
    refused(q, k, v, rows=rows, bias=attention.RelativeBias(table, max_distance=1025))
    refused(q, k, v, rows=rows, bias=attention.RelativeBias(table), q_start=torch.zeros(2, device="cuda"))
    refused(q, k, v, rows=rows, bias=attention.RelativeBias(table), q_start=1 << 30)
    out, lse = attention.attend(q, k, v, rows=rows, return_lse=True)
    with pytest.raises(vk.VkInvalidArgument):
        attention.attend_backward(q[:1], q, k, v, out, lse, rows=rows)
    with pytest.raises(vk.VkInvalidArgument):
        attention.attend_backward(q, q, k, v, out, lse[:, :, :, :1], rows=rows)
