"""The paged K/V cache on the card against a float64 restatement (oracle/paged_oracle.py).

Tolerances.  bf16 rounds to half a step, 2^-8 relative; e4m3 to 2^-4, below 2^-6 of a scale to 2^-10 of it.  An attention output differs from
the exact one by its own rounding (2^-8 |o|), by the rounding of the weights to bf16 (2^-8 of sum_j p_j |v_j|), by fp32 sums of up to some
thousand terms (2^-14 of the same, generously) and, by the factor e^(2d) - 1, by an error d of the logits.  Without norm and rotation the
operands are exact and d is the fp32 error of 128 products and the exponent, below 2^-14 for the logits here (|s| < 64).  With them
the kernel rounds a query element to bf16 as the oracle does, but from an fp32 value: where that lies within 2^-20 of a border between two bf16
numbers the two may differ by a step, 2^-7 |q|.  That happens to an element with probability 2^-12; four of a row's 128 are allowed for.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

D = 128
EPS = 1e-6
BF16 = 2.0 ** -8


def _oracle():
    from oracle import paged_oracle as P

    return P


def _rows(gen, n, heads, std=1.0):
    return (torch.randn((n, heads, D), generator=gen) * std).to(torch.bfloat16)


def _tables(gen, n):
    angle = torch.rand((n, D // 2), generator=gen, dtype=torch.float64) * 60.0 - 30.0
    return angle.cos().float(), angle.sin().float()


def _dev(t):
    if t is None:
        return None
    return tuple(x.cuda() for x in t) if isinstance(t, tuple) else t.cuda()


class Held:
    """A pool on the card and, sequence by sequence, the rows (bf16, on the host) that went into it unchanged."""

    width = 0   # least width of the tables of its batches, in pages (behind a sequence's own: none)

    def __init__(self, lengths, heads, fp8, seed=0, poison=True, std=1.0, spare=3):
        import pika_h3_flex_amd as pk

        P = _oracle()
        gen = torch.Generator().manual_seed(seed)
        pages, self.lists = P.page_lists(lengths, spare, gen)
        self.cache = pk.PagedKV(max(pages, 1), heads, fp8=fp8, device="cuda")
        if poison:   # what no sequence holds is NaN in every reading of its bytes
            self.cache.data.fill_(0xFF)
        self.lengths, self.heads, self.fp8 = list(lengths), heads, fp8
        self.k = [_rows(gen, n, heads, std) for n in lengths]
        self.v = [_rows(gen, n, heads, std) for n in lengths]
        if sum(lengths):
            pk.paged_write(self.cache, self.batch(lengths), torch.cat(self.k).cuda(), torch.cat(self.v).cuda())

    def batch(self, rows, lengths=None):
        import pika_h3_flex_amd as pk

        lists = [own + [-1] * (Held.width - len(own)) for own in self.lists]
        made = pk.PagedBatch.build(rows, self.lengths if lengths is None else lengths, self.lists, device="cuda")
        table = torch.tensor([x + [-1] * (max(1, max(map(len, lists))) - len(x)) for x in lists], dtype=torch.int32, device="cuda")
        return pk.PagedBatch(made.starts, made.lengths, table, made.rows)

    def stored(self, b):
        P = _oracle()
        return P.stored(self.k[b].double(), self.fp8), P.stored(self.v[b].double(), self.fp8)


def _check_attention(held, rows, Hq, *, causal, seed=1, norm=False, rope=0, scale=None, std=1.0, repeat=True, on="cpu", missing=(), rounded=True):
    """New rows over a cache against the oracle (run on device ``on``), every row and head; returns the output.  ``missing``: pages (sequence, which of
    its pages) that are taken out of the table.  ``rounded``: queries go to bf16 after norm and rotation."""
    import pika_h3_flex_amd as pk

    P = _oracle()
    gen = torch.Generator().manual_seed(seed)
    T = sum(rows)
    q = _rows(gen, T, Hq, std)
    w = (1.0 + 0.2 * torch.randn(D, generator=gen)) if norm else None
    tables = _tables(gen, T) if rope else None
    batch = held.batch(rows)
    for b, page in missing:
        batch.table[b, page] = -1
    opts = dict(causal=causal, q_norm_weight=_dev(w), norm_eps=EPS, rope_mode=rope, rope_q=_dev(tables), softmax_scale=scale)
    out = pk.paged_attention(q.cuda(), held.cache, batch, **opts)
    torch.cuda.synchronize()
    got = out.to(on).double()
    assert torch.isfinite(got).all()
    ready = P.norm_rope(q, w, EPS, tables, rope)
    if (norm or rope) and rounded:
        ready = ready.to(torch.bfloat16).double()
    at = 0
    for b, n in enumerate(rows):
        k, v = held.stored(b)
        gone = [page for which, page in missing if which == b]
        ref, size = P.attend(ready[at:at + n].to(on), k.to(on), v.to(on), causal=causal, scale=scale, gone=gone)
        d = 2.0 ** -14
        if k.numel() and not rounded:
            # two bf16 numbers leave 2^-18 of each element, norm and rotation in fp32 less than another 2^-18
            d = d + 2.0 ** -17 * float((ready[at:at + n].abs().amax(1) @ k.abs().amax(1).t()).max()) * (scale or 1 / math.sqrt(D))
        elif (norm or rope) and k.numel():
            d = d + 4 * 2.0 ** -7 * float(ready.abs().max() * k.abs().max()) * (scale or 1 / math.sqrt(D))
        bound = BF16 * ref.abs() + (BF16 + 2.0 ** -14 + math.expm1(2 * d)) * size * (1 + BF16)
        off = (got[at:at + n] - ref).abs() - bound
        assert float(off.max() if off.numel() else 0.0) <= 0.0, (b, n, float(off.max()), float((got[at:at + n] - ref).abs().max()))
        # the sum over all elements leaves less room than the largest of them
        if ref.numel() and float(ref.norm()) > 0:
            assert float((got[at:at + n] - ref).norm() / ref.norm()) < 2 * BF16, (b, n)
        at += n
    if repeat:
        again = pk.paged_attention(q.cuda(), held.cache, batch, **opts)
        assert torch.equal(again, out)
    return out


@pytest.fixture(params=["narrow", "wide"])
def table_width(request):
    """A call's form goes by the width of its table, which stands for the lengths: over a wide one chunks take the form of many rows, however few there are."""
    Held.width = 0 if request.param == "narrow" else 8300
    yield
    Held.width = 0


# ---- writing and reading ----

@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lengths,heads", [([1], 1), ([64], 2), ([65, 1, 130], 3), ([0, 63, 200, 0, 7], 8), ([1000, 321], 24)])
def test_rows_come_back_as_they_are_held(lengths, heads, fp8):
    import pika_h3_flex_amd as pk

    held = Held(lengths, heads, fp8, seed=len(lengths) + heads)
    k, v = pk.paged_read(held.cache, held.batch(lengths))
    want = [held.stored(b) for b in range(len(lengths))]
    assert torch.equal(k.cpu().double(), torch.cat([w[0] for w in want]))
    assert torch.equal(v.cpu().double(), torch.cat([w[1] for w in want]))


@pytest.mark.parametrize("fp8", [False, True])
def test_rows_arrive_in_pieces_and_nothing_else_is_touched(fp8):
    """Chunks of 1 to 100 rows, page by page, equal one write of everything; the pool outside of the written places keeps its bytes."""
    import pika_h3_flex_amd as pk

    lengths, heads = [150, 37, 64, 0], 3
    whole = Held(lengths, heads, fp8, seed=5, poison=False)
    whole.cache.data.fill_(0x5A)
    pk.paged_write(whole.cache, whole.batch(lengths), torch.cat(whole.k).cuda(), torch.cat(whole.v).cuda())
    pieces = pk.PagedKV(whole.cache.pages, heads, fp8=fp8, device="cuda")
    pieces.data.fill_(0x5A)
    have = [0] * 4
    for step in ([1, 1, 5, 0], [3, 0, 59, 0], [60, 20, 0, 0], [1, 16, 0, 0], [85, 0, 0, 0]):
        have = [h + n for h, n in zip(have, step)]
        cut = lambda rows: torch.cat([x[h - n:h] for x, h, n in zip(rows, have, step)]).cuda()   # noqa: E731
        pk.paged_write(pieces, whole.batch(step, have), cut(whole.k), cut(whole.v))
    assert have == lengths
    assert torch.equal(pieces.data, whole.cache.data)
    untouched = sorted(set(range(whole.cache.pages)) - {p for x in whole.lists for p in x})
    assert untouched and bool((pieces.data[untouched] == 0x5A).all())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("norm,rope", [(True, 0), (False, 1), (True, 2), (True, 1)])
def test_norm_and_rotation_of_the_keys(norm, rope, fp8):
    import pika_h3_flex_amd as pk

    P = _oracle()
    lengths, rows, heads = [100, 333], [70, 129], 5
    held = Held(lengths, heads, fp8, seed=9)
    gen = torch.Generator().manual_seed(2)
    T = sum(rows)
    wide = torch.randn((T, heads + 2, 3 * D), generator=gen).to(torch.bfloat16)
    wide_dev = wide.cuda()
    k, v = wide[:, 1:1 + heads, D:2 * D], wide[:, :heads, 2 * D:]        # strided rows
    w = (1.0 + 0.2 * torch.randn(D, generator=gen)) if norm else None
    tables = _tables(gen, T) if rope else None
    batch = held.batch(rows)
    pk.paged_write(held.cache, batch, wide_dev[:, 1:1 + heads, D:2 * D], wide_dev[:, :heads, 2 * D:], k_norm_weight=_dev(w), norm_eps=EPS,
                   rope_mode=rope, rope_k=_dev(tables))
    got_k, got_v = (t.cpu().double() for t in pk.paged_read(held.cache, batch))
    assert torch.equal(got_v, P.stored(v.double(), fp8))
    exact = P.norm_rope(k, w, EPS, tables, rope)
    slack = 2.0 ** -20 * exact.abs().amax(-1, keepdim=True)               # fp32 norm, weights and rotation
    if fp8:
        # a scale at a power of two may fall on either side of it: twice its share of the smallest step
        bound = 2.0 ** -4 * exact.abs() + 2 * 2.0 ** -10 * P.key_scales(exact) + slack
    else:
        bound = BF16 * exact.abs() + slack
    assert bool(((got_k - exact).abs() <= bound).all())
    want = P.stored(exact, fp8)
    assert float((got_k != want).double().mean()) < 2.0 ** -9              # nearly all round the same way


def test_eight_bit_rows_of_every_size():
    """Scales from the smallest to the largest that a bf16 row can need, rows of zeros, single values, magnitudes that are a power of two times 448."""
    import pika_h3_flex_amd as pk

    P = _oracle()
    gen = torch.Generator().manual_seed(3)
    n = 256
    x = torch.randn((n, 1, D), generator=gen) * torch.exp2(torch.linspace(-100, 110, n))[:, None, None]
    x[5] = 0.0
    x[6] = 0.0
    x[6, 0, 77] = 448.0
    x[7, 0] = 448.0 * 2.0 ** -3
    x[8, 0, :] = 0.0
    x[8, 0, 3] = -450.0
    x[9] = 1.0
    x = x.to(torch.bfloat16)
    held = Held([n], 1, True)
    batch = held.batch([n])
    pk.paged_write(held.cache, batch, x.cuda(), x.flip(0).contiguous().cuda())
    k, v = (t.cpu().double() for t in pk.paged_read(held.cache, batch))
    assert torch.equal(k, P.stored(x.double(), True)) and torch.equal(v, P.stored(x.flip(0).double(), True))


def test_what_is_not_finite_is_stored_as_nan():
    import pika_h3_flex_amd as pk

    P = _oracle()
    held = Held([5], 2, True)
    x = _rows(torch.Generator().manual_seed(1), 5, 2)
    bad = x.clone()
    bad[1, 0, 3], bad[1, 0, 100], bad[2, 1, 0] = float("inf"), float("nan"), float("-inf")
    pk.paged_write(held.cache, held.batch([5]), bad.cuda(), bad.cuda())
    ref = x.double()
    ref[1, 0, 3] = ref[1, 0, 100] = ref[2, 1, 0] = 0.0
    want = P.stored(ref, True)
    want[1, 0, 3] = want[1, 0, 100] = want[2, 1, 0] = float("nan")
    for got in pk.paged_read(held.cache, held.batch([5])):
        assert torch.equal(got.cpu().double().nan_to_num(1e9), want.nan_to_num(1e9))


# ---- attention ----

@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("lengths,kv,Hq", [([1], 1, 1), ([2, 63, 64, 65], 1, 3), ([33, 700, 1, 129], 2, 2), ([500, 0, 3000], 4, 24), ([40] * 70, 3, 6)])
def test_single_tokens(lengths, kv, Hq, fp8):
    held = Held(lengths, kv, fp8, seed=kv)
    _check_attention(held, [1] * len(lengths), Hq, causal=True)
    _check_attention(held, [1] * len(lengths), Hq, causal=False, norm=True, rope=1)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("rows", [[1, 1], [3, 5]])
@pytest.mark.parametrize("norm,rope", [(True, 0), (True, 1), (False, 2)])
def test_few_rows_keep_what_the_rounding_of_their_queries_leaves(rows, norm, rope, fp8):
    """Logits of +-30 and more, in which a query rounded to bf16 is off by several hundredths."""
    held = Held([500, 900], 2, fp8, seed=2, std=8.0)
    _check_attention(held, rows, 4, causal=False, norm=norm, rope=rope, rounded=False)


@pytest.mark.usefixtures("table_width")
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("rows,lengths,kv,Hq", [
    ([2, 17], [2, 100], 2, 2), ([16, 0, 33, 1], [16, 64, 64, 300], 1, 5), ([65, 5], [200, 4], 2, 6), ([200, 31], [777, 31], 3, 3),
    ([1, 300], [1500, 900], 2, 16), ([20, 20, 20], [0, 3, 500], 2, 2), ([700], [700], 1, 4)])
def test_chunks(rows, lengths, kv, Hq, causal, fp8):
    """Ragged chunks, more rows than keys, sequences without rows or keys, lengths at and around the ends of pages."""
    held = Held(lengths, kv, fp8, seed=sum(rows))
    _check_attention(held, rows, Hq, causal=causal)


@pytest.mark.usefixtures("table_width")
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("norm,rope,scale", [(True, 0, None), (False, 2, None), (True, 1, 0.05), (False, 0, 0.2)])
def test_queries_through_norm_and_rotation(norm, rope, scale, fp8):
    held = Held([300, 40, 129], 2, fp8, seed=4)
    for rows in ([1, 1, 1], [40, 7, 100]):
        _check_attention(held, rows, 4, causal=True, norm=norm, rope=rope, scale=scale)


@pytest.mark.usefixtures("table_width")
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("rows", [[1, 1], [50, 130]])
def test_large_logits_raise_the_running_maximum(rows, fp8):
    """Logits up to +-60, larger ones towards the end of the keys: the maximum is raised over and over."""
    import pika_h3_flex_amd as pk

    held = Held([900, 400], 2, fp8, seed=8, std=1.0)
    for b in range(2):
        held.k[b] = (held.k[b].float() * torch.linspace(0.1, 1.5, held.lengths[b])[:, None, None]).to(torch.bfloat16)
    pk.paged_write(held.cache, held.batch(held.lengths), torch.cat(held.k).cuda(), torch.cat(held.v).cuda())
    _check_attention(held, rows, 4, causal=False, std=8.0)


@pytest.mark.usefixtures("table_width")
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("rows,Hq", [(1, 1), (20, 1), (60, 2), (450, 1)])
@pytest.mark.parametrize("order", [1, -1])
def test_logits_that_run_over_hundreds(rows, Hq, order, fp8):
    """Keys along the queries, their logits from -200 to 200 (in powers of two: +-290) or the other way round: weights of whole tiles vanish beside those
    of others, before or after them; all queries see their last or first keys alone in the end."""
    import pika_h3_flex_amd as pk

    P = _oracle()
    n = 1000
    held = Held([n], 1, fp8, seed=3)
    gen = torch.Generator().manual_seed(1)
    direction = torch.where(torch.rand(D, generator=gen) < 0.5, -1.0, 1.0)
    ramp = torch.linspace(-200.0, 200.0, n)[::1] if order == 1 else torch.linspace(200.0, -200.0, n)
    # q k / sqrt(D) = 8 * D * x / sqrt(D) with x = ramp / (8 sqrt(D)); every component of a key has the same size, so its e4m3 value is that of x
    held.k[0] = ((ramp / (8 * math.sqrt(D)))[:, None, None] * direction).to(torch.bfloat16)
    pk.paged_write(held.cache, held.batch([n]), held.k[0].cuda(), held.v[0].cuda())
    q = (8.0 * direction).expand(rows, Hq, D).to(torch.bfloat16)
    got = pk.paged_attention(q.cuda(), held.cache, held.batch([rows])).cpu().double()
    k, v = held.stored(0)
    ref, size = P.attend(q, k, v, causal=False)
    # products are exact (q is a power of two), sums and exponents are fp32 of up to 290: 2^-23 * 290 * a few
    bound = BF16 * ref.abs() + (BF16 + math.expm1(2 * 2.0 ** -10)) * size
    assert torch.isfinite(got).all() and bool(((got - ref).abs() <= bound).all()), float((got - ref).abs().max())


def _sweep(seed):
    gen = torch.Generator().manual_seed(seed)
    pick = lambda *x: x[int(torch.randint(len(x), (1,), generator=gen))]   # noqa: E731
    size = lambda lo, hi: int(round(math.exp(float(torch.rand(1, generator=gen)) * math.log(hi / lo)) * lo))   # noqa: E731
    B, kv = pick(1, 1, 2, 3, 7), pick(1, 2, 3, 4)
    Hq = kv * pick(1, 1, 2, 5, 8)
    top = pick(1, 40, 400, 1500)
    lengths = [pick(0, size(1, 300), size(1, 9000)) if B > 1 else size(1, 20000) for _ in range(B)]
    rows = [pick(0, size(1, top), size(1, top)) if B > 1 else size(1, top) for _ in range(B)]
    missing = []
    if pick(0, 0, 1):
        missing = [(b, int(torch.randint(n // 64 + 1, (1,), generator=gen)) % ((n + 63) // 64)) for b, n in enumerate(lengths) if n for _ in range(3)]
    if not any(rows):
        rows[0] = 3
    return dict(lengths=lengths, rows=rows, kv=kv, Hq=Hq, causal=bool(pick(0, 1)), norm=bool(pick(0, 1)), rope=pick(0, 1, 2), fp8=bool(pick(0, 1)), missing=missing)


@pytest.mark.usefixtures("table_width")
@pytest.mark.parametrize("seed", range(60))
def test_random_batches(seed):
    """Seeded: ragged batches of one to seven sequences, every form of the kernel, pages taken out of the table, against the oracle on the card."""
    c = _sweep(seed)
    held = Held(c["lengths"], c["kv"], c["fp8"], seed=seed)
    _check_attention(held, c["rows"], c["Hq"], causal=c["causal"], seed=seed + 100, norm=c["norm"], rope=c["rope"], on="cuda", missing=c["missing"])


@pytest.mark.parametrize("fp8", [False, True])
def test_short_tables_under_many_rows(fp8):
    """Tables of a few pages and rows enough for every workgroup: units are not cut, and there is no second launch."""
    held = Held([70, 300, 1000, 512, 0], 8, fp8, seed=6)
    _check_attention(held, [450, 900, 1400, 30, 2], 8, causal=False, on="cuda", norm=True, rope=2)
    _check_attention(held, [90, 200, 640, 512, 70], 16, causal=True, on="cuda")


def test_long_contexts_are_shared_out():
    """Few units of many tiles: every workgroup has a part of one, and the parts are joined."""
    held = Held([9000, 20000], 2, False, seed=3)
    _check_attention(held, [1, 1], 2, causal=True)
    _check_attention(held, [3, 20], 4, causal=True)
    _check_attention(Held([20000], 1, True, seed=3), [2], 8, causal=True)


@pytest.mark.usefixtures("table_width")
@pytest.mark.parametrize("fp8", [False, True])
def test_long_units_of_many_rows_are_shared_out(fp8):
    """Units many times as long as a workgroup's run: runs inside a unit start in their middle, runs over a unit's end do the next one first; blocks with
    rows for one, two and three waves a SIMD."""
    held = Held([30000, 9000], 3, fp8, seed=3)
    for rows in ([770, 130], [300, 0]):
        _check_attention(held, rows, 3, causal=False, on="cuda", norm=True, rope=1)
    _check_attention(held, [400, 200], 6, causal=True, on="cuda")


@pytest.mark.parametrize("fp8", [False, True])
def test_more_than_64_blocks_of_a_causal_sequence(fp8):
    """Their sums are a wave's work, their places found 64 at a time; tables of more than 16 pages, so that units are cut.  Blocks of 384 rows, of 32 rows, and of
    16 rows (one long chunk among 200 sequences without rows)."""
    held = Held([3000], 1, fp8, seed=4)
    _check_attention(held, [1700], 16, causal=True, on="cuda", norm=True, rope=1)
    _check_attention(held, [150], 16, causal=True, on="cuda")
    lengths = [0] * 200
    lengths[77] = 1500
    rows = [0] * 200
    rows[77] = 1100
    _check_attention(Held(lengths, 1, fp8, seed=4), rows, 1, causal=True, on="cuda")


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("wide", [0, 40])
def test_as_many_sequences_as_a_call_takes(fp8, wide):
    """1,024 of them, some without rows, some without keys, some without either: read back as written, single tokens, ragged chunks."""
    import pika_h3_flex_amd as pk

    gen = torch.Generator().manual_seed(11)
    B = 1024
    draw = lambda hi: (torch.randint(0, hi, (B,), generator=gen) * (torch.rand(B, generator=gen) < 0.8)).tolist()   # noqa: E731
    lengths = draw(200)
    Held.width = wide
    try:
        held = Held(lengths, 1, fp8, seed=5)
        got = pk.paged_read(held.cache, held.batch(lengths))
        want = [held.stored(b) for b in range(B)]
        assert all(torch.equal(got[i].cpu().double(), torch.cat([w[i] for w in want])) for i in range(2))
        _check_attention(held, draw(2), 2, causal=True, on="cuda", repeat=False)
        _check_attention(held, draw(90), 1, causal=True, on="cuda")
        _check_attention(held, draw(90), 2, causal=False, on="cuda", norm=True, repeat=False)
    finally:
        Held.width = 0


@pytest.mark.usefixtures("table_width")
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("side", ["key", "value"])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("rows", [[3, 5], [60, 30], [500, 450]])
def test_what_is_not_finite_in_the_cache(rows, what, side, fp8):
    """One element of one key or value: rows that see it, of heads that read it, show it; no other row, head or sequence does, but where it is a value, and there
    in its column, rows of its sequence in front of it under the causal limit.  (An infinite key is NaN in 8 bits; in bf16 it gives logits of one sign a row: +inf shows, -inf is
    a key without weight.)"""
    import pika_h3_flex_amd as pk

    P = _oracle()
    lengths, at, column = [700, 600], 500, 37                               # key 500 of the first sequence, of kv head 1
    held = Held(lengths, 2, fp8, seed=21)
    bad = [torch.cat(x).clone() for x in (held.k, held.v)]
    bad[0 if side == "key" else 1][at, 1, column] = what
    pk.paged_write(held.cache, held.batch(lengths), *(t.cuda() for t in bad))
    q = _rows(torch.Generator().manual_seed(1), sum(rows), 4).cuda()
    clean = []
    for b in range(2):
        k, v = held.stored(b)
        if b == 0 and fp8:   # what is not finite counts as nothing for its row's scale: the other elements are as if it were zero
            for t, which in ((k, "key"), (v, "value")):
                if which == side:
                    row = (held.k if side == "key" else held.v)[0][at, 1].double().clone()
                    row[column] = 0.0
                    t[at, 1] = P.stored(row[None, None], True)[0, 0]
        clean.append((k.cuda(), v.cuda()))
    for causal in (False, True):
        got = pk.paged_attention(q, held.cache, held.batch(rows), causal=causal).double()
        first = 0
        for b, n in enumerate(rows):
            mine = slice(first, first + n)
            ref, size = P.attend(q[mine], *clean[b], causal=causal)
            ok = (got[mine] - ref).abs() <= BF16 * ref.abs() + (BF16 + 2.0 ** -14 + math.expm1(2 * 2.0 ** -14)) * size * (1 + BF16)
            reads = torch.zeros((n, 4, D), dtype=torch.bool, device="cuda")
            sees = torch.arange(n, device="cuda") + (lengths[b] - n) >= at if causal else torch.ones(n, dtype=torch.bool, device="cuda")
            if b == 0:
                reads[sees, 2:] = True                                      # query heads 2 and 3 read kv head 1
            if side == "value":
                may = reads.clone()
                may[:, 2:] |= causal and b == 0
                others = [c for c in range(D) if c != column]
                assert bool(ok[..., others].all()) and bool(ok[..., column][~may[..., column]].all())
                assert not bool(torch.isfinite(got[mine][..., column][reads[..., column]]).any())
            elif fp8 or math.isnan(what):
                assert bool(ok[~reads].all()) and bool(torch.isnan(got[mine][reads]).all())
            else:
                sign = torch.sign(q[mine, :, column].double() * what)[..., None].expand(n, 4, D)
                assert bool(ok[~reads].all()) and bool(torch.isnan(got[mine][reads & (sign >= 0)]).all())
                if b == 0 and not causal:
                    k, v = (torch.cat([t[:at], t[at + 1:]]) for t in clean[0])
                    ref, size = P.attend(q[mine], k, v, causal=False)
                    off = (got[mine] - ref).abs() - (BF16 * ref.abs() + (BF16 + 2.0 ** -14 + math.expm1(2 * 2.0 ** -14)) * size * (1 + BF16))
                    assert float(off[reads & (sign < 0)].max()) <= 0.0
            first += n


@pytest.mark.parametrize("fp8", [False, True])
def test_pages_that_are_not_there(fp8):
    """Table entries outside of the pool: their keys are seen by nobody, writes to them dropped, reads of them zero; the rest as without them."""
    import pika_h3_flex_amd as pk

    P = _oracle()
    lengths, kv = [200, 70], 2
    held = Held(lengths, kv, fp8, seed=6)
    rows = [5, 3]
    batch = held.batch(rows)
    table = batch.table.clone()
    table[0, 1], table[1, 0] = held.cache.pages, -5
    batch = pk.PagedBatch(batch.starts, batch.lengths, table, batch.rows)
    q = _rows(torch.Generator().manual_seed(1), 8, 4)
    got = pk.paged_attention(q.cuda(), held.cache, batch).cpu().double()
    k0, v0 = held.stored(0)
    k1, v1 = held.stored(1)
    here = [i for i in range(200) if not 64 <= i < 128]
    ref = torch.cat([P.attend(q[:5], k0[here], v0[here], causal=False)[0], P.attend(q[5:], k1[64:], v1[64:], causal=False)[0]])
    size = torch.cat([P.attend(q[:5], k0[here], v0[here], causal=False)[1], P.attend(q[5:], k1[64:], v1[64:], causal=False)[1]])
    assert bool(((got - ref).abs() <= BF16 * ref.abs() + (BF16 + 2.0 ** -12) * size).all())
    everything = pk.PagedBatch.build(lengths, lengths, held.lists, device="cuda")
    everything.table.copy_(table)
    k, v = pk.paged_read(held.cache, everything)
    want = torch.cat([k0, k1])
    want[64:128] = 0
    want[200:264] = 0
    assert torch.equal(k.cpu().double(), want) and bool((v[64:128] == 0).all()) and bool((v[200:264] == 0).all())
    before = held.cache.data.clone()
    table.fill_(2 ** 31 - 1)
    nowhere = pk.PagedBatch(everything.starts, everything.lengths, table, everything.rows)
    pk.paged_write(held.cache, nowhere, torch.cat(held.k).cuda(), torch.cat(held.v).cuda())
    assert torch.equal(held.cache.data, before)
    assert bool((pk.paged_attention(q.cuda(), held.cache, pk.PagedBatch(batch.starts, batch.lengths, table, 8)) == 0).all())


def test_arrays_out_of_range_are_brought_into_it():
    """starts beyond the rows, lengths beyond the table: as the header says, and rows of no sequence keep what they held."""
    import pika_h3_flex_amd as pk

    held = Held([128, 64], 2, False, seed=6)
    q = _rows(torch.Generator().manual_seed(1), 6, 2).cuda()
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    table = held.batch([0, 0]).table
    wild = pk.PagedBatch(as_int([1, 4, 99]), as_int([10 ** 9, -3]), table)
    tame = pk.PagedBatch(as_int([1, 4, 6]), as_int([128, 0]), table)
    a, b = (torch.full_like(q, 7.0) for _ in range(2))
    pk.paged_attention(q, held.cache, wild, out=a)
    pk.paged_attention(q, held.cache, tame, out=b)
    assert torch.equal(a, b) and bool((a[0] == 7.0).all()) and bool((a[4:] == 0).all())
    ka, va = (torch.full((6, 2, D), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pk.paged_read(held.cache, wild, out=(ka, va))
    assert bool((ka[0] == 7.0).all()) and bool((ka[4:] == 0).all()) and torch.equal(ka[1:4].cpu(), held.k[0][125:128])
    backwards = pk.PagedBatch(as_int([4, 1, 1]), as_int([128, 64]), table)
    c = torch.full_like(q, 7.0)
    pk.paged_attention(q, held.cache, backwards, out=c)
    assert bool((c == 7.0).all())


@pytest.mark.parametrize("fp8", [False, True])
def test_a_write_past_the_table_leaves_what_is_stored(fp8):
    """Tokens behind the last place of their table, and sequences that say they have rows the call does not: no stored byte changes but those of rows in
    their own place."""
    import pika_h3_flex_amd as pk

    held = Held([128, 64], 2, fp8, seed=6)
    table = held.batch([0, 0]).table.clone()
    table[1, 1] = table[0, 0]                                              # a page that both hold
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    gen = torch.Generator().manual_seed(2)
    k, v = (_rows(gen, 6, 2).cuda() for _ in range(2))
    before = held.cache.data.clone()
    for starts, lengths in (([0, 1, 2], [129, 129]), ([0, 3, 6], [10 ** 9, 2 ** 31 - 1]), ([0, 0, 99], [0, -3]), ([2, 6, 6], [132, 0]),
                            ([-9, 0, 6], [128, -2 ** 31]), ([0, 2 ** 31 - 1, 6], [-5, 0])):
        pk.paged_write(held.cache, pk.PagedBatch(as_int(starts), as_int(lengths), table), k, v)
        assert torch.equal(held.cache.data, before), (starts, lengths)
    # four rows up to one behind the table: three in their place; eight rows of which the call has six, and of these one is in front of position 0
    for starts, lengths, where in (([1, 5, 5], [129, 0], (0, 1, 4, 125)), ([0, 0, 8], [0, 7], (1, 1, 6, 0))):
        pk.paged_write(held.cache, pk.PagedBatch(as_int(starts), as_int(lengths), table), k, v)
        b, lo, hi, first = where
        twin = pk.PagedKV(held.cache.pages, 2, fp8=fp8, data=before.clone())
        keys = [0, 0]
        keys[b] = first + hi - lo
        pk.paged_write(twin, pk.PagedBatch(as_int([0, 0 if b else hi - lo, hi - lo]), as_int(keys), table), k[lo:hi], v[lo:hi])
        assert torch.equal(held.cache.data, twin.data) and not torch.equal(twin.data, before)
        held.cache.data.copy_(before)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("rows,wide", [(4, 0), (30, 0), (130, 0), (130, 8000)])
def test_a_causal_chunk_over_the_end_of_its_table(rows, wide, fp8):
    """Rows whose places are behind the table, or that the call does not have, move no other row: each sees what is stored up to its own place."""
    import pika_h3_flex_amd as pk

    P = _oracle()
    held = Held([320, 64], 2, fp8, seed=6)
    table = held.batch([0, 0]).table
    stored = [t.cuda() for t in held.stored(0)]
    table = torch.cat([table, table.new_full((2, wide), -1)], 1)                         # (another form over a wide table, whose pages are not there)
    q = _rows(torch.Generator().manual_seed(1), rows, 4).cuda()
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")                 # noqa: E731
    for end, length in ((rows, 320 + rows // 2), (rows, 320 + 2 * rows), (rows + 3, 300), (rows + 40, 350), (rows, 10 ** 9), (rows, rows // 2)):
        batch = pk.PagedBatch(as_int([0, end, end]), as_int([length, 0]), table)
        got = pk.paged_attention(q, held.cache, batch, causal=True).double()
        own = length - end + torch.arange(rows)                                          # the rows' places
        for r in {0, 1, rows // 2, rows - 1}:
            m = max(0, min(320, length, int(own[r]) + 1))
            ref, size = P.attend(q[r:r + 1], stored[0][:m], stored[1][:m], causal=False)
            bound = BF16 * ref.abs() + (BF16 + 2.0 ** -14 + math.expm1(2 * 2.0 ** -14)) * size * (1 + BF16)
            assert bool(((got[r:r + 1] - ref).abs() <= bound).all()), (end, length, r)


def test_strides_order_and_the_output_in_the_queries_place():
    import pika_h3_flex_amd as pk

    held = Held([300, 90], 2, False, seed=7)
    batch = held.batch([40, 3])
    gen = torch.Generator().manual_seed(5)
    q = _rows(gen, 43, 6).cuda()
    want = pk.paged_attention(q, held.cache, batch, causal=True)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)           # [rows, heads, 128] with the heads outermost in memory
    wide = torch.full((43, 6, 2 * D), 3.0, dtype=torch.bfloat16, device="cuda")
    got = pk.paged_attention(heads_first, held.cache, batch, causal=True, out=wide[..., D:])
    assert torch.equal(got, want) and bool((wide[..., :D] == 3.0).all())
    same = q.clone()
    assert torch.equal(pk.paged_attention(same, held.cache, batch, causal=True, out=same), want)
    table = torch.full((2, 40), -1, dtype=torch.int32, device="cuda")[:, ::1]
    table[:, :batch.table.shape[1]] = batch.table
    assert torch.equal(pk.paged_attention(q, held.cache, pk.PagedBatch(batch.starts, batch.lengths, table[:, :batch.table.shape[1] + 3]), causal=True), want)


def test_one_page_in_two_sequences():
    """A prefix that two sequences share is read by both."""
    import pika_h3_flex_amd as pk

    P = _oracle()
    held = Held([64 + 20, 64 + 50], 1, False, seed=2)
    lists = [list(x) for x in held.lists]
    lists[1][0] = lists[0][0]
    batch = pk.PagedBatch.build([1, 1], held.lengths, lists, device="cuda")
    q = _rows(torch.Generator().manual_seed(1), 2, 1)
    got = pk.paged_attention(q.cuda(), held.cache, batch).cpu().double()
    (k0, v0), (k1, v1) = held.stored(0), held.stored(1)
    ref, size = P.attend(q[1:], torch.cat([k0[:64], k1[64:]]), torch.cat([v0[:64], v1[64:]]), causal=False)
    assert bool(((got[1:] - ref).abs() <= BF16 * ref.abs() + (BF16 + 2.0 ** -12) * size).all())


def test_rows_of_no_sequence_are_zeros_in_new_outputs():
    """A padded batch (rows in front of the first sequence and behind the last, their number not known to the host): new outputs hold zeros there, given ones
    what they held, eager, captured and through the processor."""
    import pika_h3_flex_amd as pk

    held = Held([300, 64, 5], 2, False, seed=3)
    made = held.batch([4, 0, 2])
    batch = pk.PagedBatch(made.starts + 3, made.lengths, made.table)       # rows 3 .. 8 of 40
    q = _rows(torch.Generator().manual_seed(1), 40, 4).cuda()
    ours, rest = slice(3, 9), [i for i in range(40) if not 3 <= i < 9]

    def used():   # memory of the sizes that the calls will ask for has been used before
        for n in (4, 2, 2):
            torch.full((40, n, D), 7.0, dtype=torch.bfloat16, device="cuda")

    def calls():
        return [pk.paged_attention(q, held.cache, batch), *pk.paged_read(held.cache, batch, 40)]

    given = [torch.full((40, n, D), 7.0, dtype=torch.bfloat16, device="cuda") for n in (4, 2, 2)]
    pk.paged_attention(q, held.cache, batch, out=given[0])
    pk.paged_read(held.cache, batch, out=given[1:])
    assert all(bool((t[rest] == 7.0).all()) for t in given)
    used()
    for t, want in zip(calls(), given):
        assert torch.equal(t[ours], want[ours]) and bool((t[rest] == 0).all())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = calls()
    for _ in range(3):
        for t in got:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        for t, want in zip(got, given):
            assert torch.equal(t[ours], want[ours]) and bool((t[rest] == 0).all())
    mod = _Module(4, 2, 256, 3).cuda()
    x = torch.randn((1, 40, 256), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    with torch.no_grad():
        used()
        y = pk.PikaH3AttnProcessor()(mod, x, paged_kv=held.cache, paged_batch=batch, paged_write=False)
    assert bool((y[0, rest] == 0).all()) and bool(y[0, ours].any(-1).all())


def test_calls_follow_tensors_that_moved():
    """Lengths, table and pool given other memory, other sizes and other strides between two calls: the next one is that of a batch made of them anew."""
    import pika_h3_flex_amd as pk

    held = Held([100, 63], 2, False, seed=1)
    batch, cache = held.batch([3, 2]), held.cache
    q = _rows(torch.Generator().manual_seed(1), 5, 4).cuda()
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731

    def same():
        fresh = pk.PagedBatch(*(t.clone() for t in (batch.starts, batch.lengths, batch.table)), batch.rows)
        pool = pk.PagedKV(cache.pages, 2, data=cache.data.clone())
        got, want = (pk.paged_attention(q, c, b, causal=True) for c, b in ((cache, batch), (pool, fresh)))
        return torch.equal(got, want) and bool(torch.isfinite(got).all()) and bool(got.any())

    assert same()
    batch.lengths.data = as_int([50, 13])
    assert same()
    batch.table.set_(torch.cat([batch.table, torch.full((2, 7), -1, dtype=torch.int32, device="cuda")], 1)[:, :4])
    assert same()
    before = cache.data.detach()
    cache.data.data = before.clone()
    before.zero_()
    assert same()
    batch.lengths.resize_(1)
    with pytest.raises(ValueError, match="starts"):
        pk.paged_attention(q, cache, batch, causal=True)
    batch.starts.resize_(2), batch.table.set_(batch.table[:1].clone())
    batch.starts.copy_(as_int([0, 5]))
    assert same()


def test_a_captured_step_replays_with_changed_batches():
    """A token step in a graph: rows, lengths, pages and inputs change in place between the replays, and every replay equals the eager calls."""
    import pika_h3_flex_amd as pk

    for fp8 in (False, True):
        held = Held([100, 63, 5], 2, fp8, seed=1, spare=9)
        used = [list(x) for x in held.lists]
        free = [p for p in range(held.cache.pages) if p not in {y for x in used for y in x}]
        table = torch.full((3, 4), -1, dtype=torch.int32)
        for b, x in enumerate(used):
            x += [free.pop() for _ in range(4 - len(x))]
            table[b] = torch.tensor(x, dtype=torch.int32)
        as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
        batch = pk.PagedBatch(as_int([0, 1, 2, 3]), as_int([100, 63, 5]), table.cuda())
        gen = torch.Generator().manual_seed(4)
        q, k, v = (torch.zeros((3, h, D), dtype=torch.bfloat16, device="cuda") for h in (4, 2, 2))
        out = torch.empty_like(q)

        def step(cache, out):
            pk.paged_write(cache, batch, k, v)
            pk.paged_attention(q, cache, batch, causal=True, out=out)

        twin = pk.PagedKV(held.cache.pages, 2, fp8=fp8, data=held.cache.data.clone())
        pk.paged_attention(q, held.cache, batch, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(held.cache, out)
        for turn in range(4):
            batch.lengths.add_(as_int([1, 2, 60]) if turn == 2 else 1)
            for t, h in ((q, 4), (k, 2), (v, 2)):
                t.copy_(_rows(gen, 3, h))
            eager = torch.empty_like(q)
            step(twin, eager)
            graph.replay()
            torch.cuda.synchronize()
            # (bits: the jump of turn 2 brings keys into two of the sequences that nobody wrote, and those hold NaN)
            assert torch.equal(out.view(torch.int16), eager.view(torch.int16)) and bool(torch.isfinite(out[0 if turn >= 2 else slice(None)]).all()), turn
            assert torch.equal(held.cache.data, twin.data)


@pytest.mark.parametrize("total,Hq", [(2, 4), (40, 4), (700, 2)])
@pytest.mark.parametrize("fp8", [False, True])
def test_cuts_move_between_replays(fp8, total, Hq):
    """A table of many pages and one workspace: which units are cut, where, and how many parts they have follows rows and lengths as they are at each replay; every one
    against the oracle."""
    import pika_h3_flex_amd as pk

    P = _oracle()
    held = Held([6000, 9000], 2, fp8, seed=13)
    stored = [tuple(t.cuda() for t in held.stored(b)) for b in range(2)]
    made = held.batch([0, 0])
    batch = pk.PagedBatch(made.starts, made.lengths, made.table)
    q, out = (torch.zeros((total, Hq, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    scratch = []

    def workspace(device, n):
        if not scratch:
            scratch.append(torch.full((n,), 0xFF, dtype=torch.uint8, device=device))
        return scratch[0]

    call = lambda: pk.paged_attention(q, held.cache, batch, causal=True, out=out, workspace=workspace)   # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    gen = torch.Generator().manual_seed(total)
    for turn, (share, lengths) in enumerate([(0.5, [6000, 9000]), (1.0, [70, 4000]), (0.0, [5999, 8001]), (0.9, [6000, 1]), (0.02, [0, 9000]), (0.5, [64, 65]), (0.5, [6000, 9000])]):
        n = [round(share * total), total - round(share * total)]
        batch.starts.copy_(torch.tensor([0, n[0], total], dtype=torch.int32))
        batch.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        q.copy_(_rows(gen, total, Hq))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        at = 0
        for b in range(2):
            ref, size = P.attend(q[at:at + n[b]], stored[b][0][:lengths[b]], stored[b][1][:lengths[b]], causal=True)
            off = (out[at:at + n[b]].double() - ref).abs() - (BF16 * ref.abs() + (BF16 + 2.0 ** -14 + math.expm1(2 * 2.0 ** -14)) * size * (1 + BF16))
            assert float(off.max() if off.numel() else 0.0) <= 0.0, (turn, b)
            at += n[b]


def test_two_streams_with_a_workspace_each():
    import pika_h3_flex_amd as pk

    held = Held([5000, 3000], 4, True, seed=2)
    batch = held.batch([1, 20])
    gen = torch.Generator().manual_seed(3)
    qs = [_rows(gen, 21, 8).cuda() for _ in range(2)]
    want = [pk.paged_attention(q, held.cache, batch, causal=True) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(pk.paged_attention(qs[i], held.cache, batch, causal=True))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_a_given_workspace_may_hold_anything():
    import pika_h3_flex_amd as pk

    held = Held([4000], 2, False, seed=2)
    batch = held.batch([3])
    q = _rows(torch.Generator().manual_seed(3), 3, 2).cuda()
    want = pk.paged_attention(q, held.cache, batch)
    seen = []

    def scratch(device, nbytes):
        seen.append(nbytes)
        return torch.full((nbytes,), 0xFF, dtype=torch.uint8, device=device)

    assert torch.equal(pk.paged_attention(q, held.cache, batch, workspace=scratch), want) and seen
    small = torch.empty(16, dtype=torch.uint8, device="cuda")              # too small: the call takes one of its own
    assert torch.equal(pk.paged_attention(q, held.cache, batch, workspace=small), want)


def test_a_workspace_with_gaps_is_refused():
    """Its elements are not its bytes from the first on: what lies between them is somebody else's."""
    import pika_h3_flex_amd as pk

    held = Held([4000], 2, False, seed=2)
    q = _rows(torch.Generator().manual_seed(3), 3, 2).cuda()
    sizes = []
    pk.paged_attention(q, held.cache, held.batch([3]), workspace=lambda device, n: sizes.append(n) or torch.empty(n, dtype=torch.uint8, device=device))
    for gaps in (torch.zeros((sizes[0], 2), dtype=torch.uint8, device="cuda")[:, 0], torch.zeros(1, dtype=torch.uint8, device="cuda").expand(sizes[0])):
        with pytest.raises(ValueError, match="contiguous"):
            pk.paged_attention(q, held.cache, held.batch([3]), workspace=gaps)
        assert not bool(gaps.any())


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("new", [1, 40])
def test_offsets_past_32_bits(new, fp8):
    """Pages behind the pool's first 4 GiB, and rows more than 4 GiB apart in their tensors: written, read back and attended to as the same rows close together are."""
    import pika_h3_flex_amd as pk

    P, H = _oracle(), 24
    pages = -(-(5 << 30) // (H * int(pk._lib.load().pkh3_paged_record_bytes(pk._lib.PAGED_FP8 if fp8 else 0))))
    cache = pk.PagedKV(pages, H, fp8=fp8, device="cuda")
    lists, lengths = [[pages - 1, 0, pages - 3], [pages - 2]], [150, 64]
    gen = torch.Generator().manual_seed(4)
    k, v = (_rows(gen, sum(lengths), H) for _ in range(2))
    pk.paged_write(cache, pk.PagedBatch.build(lengths, lengths, lists, device="cuda"), k.cuda(), v.cuda())
    sk, sv = (P.stored(t.double(), fp8) for t in (k, v))
    back = pk.paged_read(cache, pk.PagedBatch.build(lengths, lengths, lists, device="cuda"))
    assert torch.equal(back[0].cpu().double(), sk) and torch.equal(back[1].cpu().double(), sv)
    q = _rows(gen, 2 * new, H)
    batch = pk.PagedBatch.build([new, new], lengths, lists, device="cuda")
    got = pk.paged_attention(q.cuda(), cache, batch)
    for b, (lo, hi) in enumerate(((0, 150), (150, 214))):
        ref, size = P.attend(q[b * new:(b + 1) * new], sk[lo:hi], sv[lo:hi], causal=False)
        off = (got[b * new:(b + 1) * new].cpu().double() - ref).abs() - (BF16 * ref.abs() + (BF16 + 2.0 ** -12) * size)
        assert float(off.max()) <= 0.0
    if new == 1:   # two rows, 2^31 + 64 elements from one to the other
        step = 2 ** 31 + 64
        far = torch.empty(step + H * D, dtype=torch.bfloat16, device="cuda").as_strided((2, H, D), (step, D, 1))
        far.copy_(q.cuda())
        assert torch.equal(pk.paged_attention(far, cache, batch), got)
        pk.paged_attention(q.cuda(), cache, batch, out=far)
        assert torch.equal(far, got)
        far.copy_(k[:2].cuda())
        ends = pk.PagedBatch.build([1, 1], lengths, lists, device="cuda")
        pk.paged_write(cache, ends, far, far)
        near = pk.paged_read(cache, ends)
        assert torch.equal(near[0].cpu().double(), sk[:2])
        far.zero_()
        pk.paged_read(cache, ends, out=(near[1], far))
        assert torch.equal(far.cpu().double(), P.stored(k[:2].double(), fp8))


def test_empty_calls():
    import pika_h3_flex_amd as pk

    held = Held([70], 2, False)
    batch = held.batch([0])
    none = torch.empty((0, 2, D), dtype=torch.bfloat16, device="cuda")
    assert pk.paged_attention(none, held.cache, batch).shape == (0, 2, D)
    pk.paged_write(held.cache, batch, none, none)
    assert pk.paged_read(held.cache, batch)[0].shape == (0, 2, D)


def test_agrees_with_attention_over_the_same_rows():
    """The paged call against the dense one of this library on the rows that paged_read gives back."""
    import pika_h3_flex_amd as pk

    for fp8 in (False, True):
        held = Held([640], 4, fp8, seed=12)
        q = _rows(torch.Generator().manual_seed(3), 200, 4).cuda()
        got = pk.paged_attention(q, held.cache, held.batch([200]))
        k, v = pk.paged_read(held.cache, held.batch([640]))
        dense = pk.attention(q[None], k[None], v[None])[0]
        # both round their weights and outputs to bf16, the dense call its queries too (after the softmax scale): logits off by at most 2^-8 |q| |k| / sqrt(D)
        size = pk.attention(q[None], k[None], v[None].abs())[0].float()
        d = 2.0 ** -8 * float(q.float().norm(dim=-1).max() * k.float().norm(dim=-1).max()) / math.sqrt(D)
        assert bool(((got.float() - dense.float()).abs() <= (4 * BF16 + math.expm1(2 * d)) * size).all())


# ---- through the attention processor ----

class _Norm(torch.nn.Module):
    def __init__(self, gen):
        super().__init__()
        self.weight = torch.nn.Parameter(1.0 + 0.1 * torch.randn(D, generator=gen))
        self.eps = EPS


class _Module(torch.nn.Module):
    """An attention module as the processor finds it: ``kv`` heads of keys and values, ``heads`` of queries."""

    def __init__(self, heads, kv, width, seed):
        super().__init__()
        gen = torch.Generator().manual_seed(seed)
        linear = lambda i, o: torch.nn.Linear(i, o, bias=False)   # noqa: E731
        self.heads = heads
        self.to_q, self.to_k, self.to_v = linear(width, heads * D), linear(width, kv * D), linear(width, kv * D)
        self.to_out = torch.nn.ModuleList([linear(heads * D, width)])
        for m in (self.to_q, self.to_k, self.to_v, self.to_out[0]):
            m.weight.data = torch.randn(m.weight.shape, generator=gen) / math.sqrt(m.weight.shape[1])
        self.to(torch.bfloat16)
        self.norm_q, self.norm_k = _Norm(gen), _Norm(gen)


@pytest.mark.parametrize("fp8", [False, True])
def test_a_document_continued_by_the_processor(fp8):
    """Frames of two documents arrive chunk by chunk through the processor; every chunk's output is that of the library's calls on the rows that the
    projections give, and without the cache's rounding the last one is that of the dense processor over the whole document."""
    import pika_h3_flex_amd as pk

    heads, kv, width = 4, 4, 256
    mod = _Module(heads, kv, width, 3).cuda()
    proc = pk.PikaH3AttnProcessor(rope_mode=pk.ROPE_INTERLEAVED)
    lists = [[3, 0, 7, 5], [1, 4, 2, 6]]
    cache, twin = pk.PagedKV(8, kv, fp8=fp8, device="cuda"), pk.PagedKV(8, kv, fp8=fp8, device="cuda")
    gen = torch.Generator().manual_seed(8)
    docs = [torch.randn((200, width), generator=gen).to(torch.bfloat16).cuda() for _ in range(2)]
    where = torch.rand((2, 200, 3), generator=gen, dtype=torch.float64).cuda() * 30.0
    have = [0, 0]
    last = None
    with torch.no_grad():
        for step in ([100, 64], [1, 1], [99, 0], [0, 135]):
            have = [h + n for h, n in zip(have, step)]
            rows = torch.cat([docs[b][have[b] - step[b]:have[b]] for b in range(2)])
            pos = torch.cat([where[b][have[b] - step[b]:have[b]] for b in range(2)])
            batch = pk.PagedBatch.build(step, have, lists, device="cuda")
            got = proc(mod, rows[None], position_ids=pos, paged_kv=cache, paged_batch=batch)
            tabs = pk.rope_tables(pos)
            heads_of = lambda x, h: x.view(len(rows), h, D)   # noqa: E731
            pk.paged_write(twin, batch, heads_of(mod.to_k(rows), kv), heads_of(mod.to_v(rows), kv), k_norm_weight=mod.norm_k.weight.detach(), norm_eps=EPS,
                           rope_mode=1, rope_k=tabs)
            o = pk.paged_attention(heads_of(mod.to_q(rows), heads), twin, batch, q_norm_weight=mod.norm_q.weight.detach(), norm_eps=EPS, rope_mode=1, rope_q=tabs)
            assert torch.equal(got[0], mod.to_out[0](o.view(len(rows), -1)))
            last = (step, got)
        if not fp8:
            b = 1
            dense = proc(mod, docs[b][None], position_ids=where[b])[0, 200 - last[0][b]:]
            # both round weights, operands and outputs to bf16 on the way: differences of bf16 size
            assert float((last[1][0].float() - dense.float()).norm() / dense.float().norm()) < 4 * BF16


def test_text_keys_of_several_requests_through_the_processor():
    """Cross-attention: text states of three requests of other lengths go into the pages once, and later steps find their keys there."""
    import pika_h3_flex_amd as pk

    heads, width = 4, 256
    mod = _Module(heads, heads, width, 5).cuda()
    proc = pk.PikaH3AttnProcessor()
    text = [77, 302, 5]
    rows = [130, 40, 64]
    gen = torch.Generator().manual_seed(2)
    states = [torch.randn((n, width), generator=gen).to(torch.bfloat16).cuda() for n in text]
    cache = pk.PagedKV(9, heads, device="cuda")
    lists = [[8, 1], [0, 3, 5, 7, 2], [6]]
    with torch.no_grad():
        proc.write_paged(mod, torch.cat(states)[None], cache, pk.PagedBatch.build(text, text, lists, device="cuda"))
        batch = pk.PagedBatch.build(rows, text, lists, device="cuda")
        for step in range(2):
            x = [torch.randn((n, width), generator=gen).to(torch.bfloat16).cuda() for n in rows]
            got = proc(mod, torch.cat(x)[None], paged_kv=cache, paged_batch=batch, paged_write=False)[0]
            want = torch.cat([proc(mod, xs[None], encoder_hidden_states=t[None])[0] for xs, t in zip(x, states)])
            assert float((got.float() - want.float()).norm() / want.float().norm()) < 4 * BF16


def test_keys_written_by_the_processor_take_their_own_norm():
    """norm_k's weight and epsilon, whatever norm_q's are."""
    import pika_h3_flex_amd as pk

    mod = _Module(2, 2, 64, 5).cuda()
    mod.norm_k.eps = 0.5
    cache, twin = (pk.PagedKV(1, 2, device="cuda") for _ in range(2))
    batch = pk.PagedBatch.build([20], [20], [[0]], device="cuda")
    x = _rows(torch.Generator().manual_seed(1), 20, 1)[:, 0, :64].contiguous().cuda()
    with torch.no_grad():
        pk.PikaH3AttnProcessor().write_paged(mod, x[None], cache, batch)
        k, v = mod.to_k(x).view(20, 2, D), mod.to_v(x).view(20, 2, D)
        pk.paged_write(twin, batch, k, v, k_norm_weight=mod.norm_k.weight.detach(), norm_eps=0.5)
        assert all(torch.equal(a, b) for a, b in zip(pk.paged_read(cache, batch), pk.paged_read(twin, batch)))
        mod.norm_k.eps = EPS
        pk.PikaH3AttnProcessor().write_paged(mod, x[None], cache, batch)
        assert not torch.equal(pk.paged_read(cache, batch)[0], pk.paged_read(twin, batch)[0])


def test_settings_of_dense_calls_do_not_reach_paged_ones():
    """fp8 QK^T, fused projections, merged adapters and kept cross-attention keys are settings of calls without pages: a paged call's result is the plain one's."""
    import pika_h3_flex_amd as pk

    mod = _Module(4, 2, 512, 3).cuda()
    x = torch.randn((1, 70, 512), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    batch = pk.PagedBatch.build([30, 40], [30, 40], [[2], [0]], device="cuda")
    got = []
    with torch.no_grad():
        for settings in (dict(), dict(fp8_qk=True), dict(fp8_qk="pow2", fused_projections=True, merge_adapters=True), dict(cache_cross_kv=True)):
            cache = pk.PagedKV(3, 2, device="cuda")
            got.append(pk.PikaH3AttnProcessor(**settings)(mod, x, paged_kv=cache, paged_batch=batch, paged_causal=True))
    assert bool(torch.isfinite(got[0]).all()) and all(torch.equal(g, got[0]) for g in got[1:])


def _grows(proc, mod, cache, batch, x, where):
    return proc(mod, x, position_ids=where, paged_kv=cache, paged_batch=batch, paged_causal=True)


@pytest.mark.parametrize("warm", [True, False])
def test_a_captured_processor_step_rotates_by_the_positions_of_each_replay(warm):
    """One token of two documents through the processor in a graph: rows, lengths and positions change in place, and every replay equals an eager step of a
    processor of its own."""
    import pika_h3_flex_amd as pk

    mod = _Module(4, 2, 256, 7).cuda()
    caches = [pk.PagedKV(6, 2, device="cuda") for _ in range(2)]
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")   # noqa: E731
    batch = pk.PagedBatch(as_int([0, 1, 2]), as_int([30, 61]), as_int([[3, 0, 5], [1, 4, 2]]))
    x = torch.zeros((1, 2, 256), dtype=torch.bfloat16, device="cuda")
    where = torch.ones((2, 3), dtype=torch.float64, device="cuda")
    proc, gen = pk.PikaH3AttnProcessor(), torch.Generator().manual_seed(8)
    for cache in caches:                                                   # what came before
        k, v = (_rows(torch.Generator().manual_seed(s), 89, 2).cuda() for s in (1, 2))
        pk.paged_write(cache, pk.PagedBatch.build([29, 60], [29, 60], [[3], [1]], device="cuda"), k, v)
    with torch.no_grad():
        x.copy_(torch.randn((1, 2, 256), generator=gen))
        _grows(proc if warm else pk.PikaH3AttnProcessor(), mod, caches[0], batch, x, where)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _grows(proc, mod, caches[0], batch, x, where)
        # an eager call of the same processor at the same positions, before any replay
        want = _grows(pk.PikaH3AttnProcessor(), mod, caches[1], batch, x, where)
        assert torch.equal(_grows(proc, mod, caches[0], batch, x, where), want)
        for turn in range(6):
            if turn:
                batch.lengths.add_(1)
            x.copy_(torch.randn((1, 2, 256), generator=gen))
            where.copy_(torch.rand((2, 3), generator=gen, dtype=torch.float64) * 40.0)
            want = _grows(pk.PikaH3AttnProcessor(), mod, caches[1], batch, x, where)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and bool(torch.isfinite(out).all()), turn
            assert all(torch.equal(a, b) for a, b in zip(pk.paged_read(caches[0], batch, 2), pk.paged_read(caches[1], batch, 2)))


def test_a_captured_processor_step_has_scratch_of_its_own():
    """What the processor keeps for its eager calls is not in the graph: a larger call that replaces it leaves the replays right, and they leave alone what has
    the memory by then."""
    import pika_h3_flex_amd as pk

    mod = _Module(4, 2, 256, 7).cuda()
    held = Held([900, 400], 2, False, seed=2)
    batch = held.batch([2, 1])
    x = torch.randn((1, 3, 256), generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).cuda()
    step = lambda b, rows: proc(mod, rows, paged_kv=held.cache, paged_batch=b, paged_write=False)   # noqa: E731
    proc = pk.PikaH3AttnProcessor()
    side = torch.cuda.Stream()
    with torch.no_grad(), torch.cuda.stream(side):
        want = step(batch, x)
        (key, small), = proc._workspaces.items()
        kept = small.numel()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = step(batch, x)
        assert list(proc._workspaces) == [key] and proc._workspaces[key] is small
        rows = torch.randn((1, 700, 256), generator=torch.Generator().manual_seed(8)).to(torch.bfloat16).cuda()
        wide = held.batch([400, 300])
        many = pk.PagedBatch(wide.starts, wide.lengths, torch.cat([wide.table, torch.full((2, 9000), -1, dtype=torch.int32, device="cuda")], 1), 700)
        del small
        step(many, rows)
        assert proc._workspaces[key].numel() > kept
        taken = [torch.full((kept,), 7, dtype=torch.uint8, device="cuda") for _ in range(4)]
        for _ in range(3):
            out.zero_()
            graph.replay()
            side.synchronize()
            assert torch.equal(out, want) and all(bool((t == 7).all()) for t in taken)
