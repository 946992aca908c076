"""The 8-bit KV cache on the GPU against its definition in 64 bits: writing
(byte for byte), reading back (exact), decode and prefill attention.

Tolerances of attention, from the roundings alone (u16 = 2^-11, half a step of
f16; ub = 2^-8, half a step of bf16), with A = sum_j p_j |v_j| / sum_j p_j:
the weights' f16 rounding moves the output by at most u16 A, what underflows in
f16 by n 2^-25 of the largest |v| / 2^8, and scores that are off by d (relative
weights off by about d) by 2 d A. d: the fp32 sum of 128 exact products, its
scaling and 2^x, at most 2^-17 of sum |q||k| * scale in log2 units plus 2^-21.
Then the output's own rounding, ub |o|."""
import pytest
import torch

from conftest import sub

pytestmark = pytest.mark.gpu

PAGE, D = 16, 128


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _bytes_of(pages):
    return pages.values.view(torch.uint8)


def _fill(pages, values, exps):
    _bytes_of(pages).copy_(values.view(torch.uint8))
    pages.exps.copy_(exps)


def _cache(lens, nkv, seed=0, columns=None, spread=0, extra=3):
    """A cache whose requests' rows are random and whose other rows are NaN
    bytes with exponent 255; (k, v, kv_len, block_table)."""
    ops, f8 = sub("ops"), sub("ops.fp8_pages")
    g = _gen(seed)
    counts = [-(-n // PAGE) for n in lens]
    blocks = sum(counts) + extra
    perm = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
    cols = columns or max(max(counts), 1)
    table = torch.full((len(lens), cols), -1, dtype=torch.int32, device="cuda")
    live = torch.zeros(blocks, PAGE, dtype=torch.bool, device="cuda")
    at = 0
    for r, n in enumerate(lens):
        mine = perm[at:at + counts[r]]
        table[r, :counts[r]] = mine
        at += counts[r]
        live[mine.long()] = torch.arange(counts[r] * PAGE, device="cuda").view(-1, PAGE) < n
    cache = ops.fp8_cache(blocks, nkv, "cuda")
    for i, c in enumerate(cache):
        x = torch.randn(blocks, nkv, PAGE, D, device="cuda", generator=g)
        if i == 0:
            x[..., ::13] *= 3
        if spread:  # rows of very different magnitude
            x *= torch.exp2(torch.randint(-spread, spread + 1, (blocks, nkv, PAGE, 1), device="cuda",
                                          generator=g).float())
        v, e = f8.quantize_rows(x)
        v = torch.where(live[:, None, :, None], v.view(torch.uint8), 0x7F)
        _fill(c, v, torch.where(live[:, None, :], e, 255))
    return cache[0], cache[1], torch.tensor(lens, dtype=torch.int32, device="cuda"), table


def _row(pages, table_row, n):
    """[n, nkv, 128] fp64 of a request."""
    ref = sub("ops.reference")
    if n == 0:
        return torch.zeros(0, pages.shape[1], D, dtype=torch.float64, device="cuda")
    return ref.gather_kv(pages, table_row, n).double()


def _attention(q, k, v, scale, last=None):
    """fp64 (output, tolerance) of q [rows, nq, 128] over k, v [n, nkv, 128];
    row i sees keys 0..last[i]."""
    G = q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    n = k.shape[0]
    if n == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    s = torch.einsum("qhd,khd->hqk", q, k) * scale
    hidden = torch.zeros(q.shape[0], n, dtype=torch.bool, device=q.device)
    if last is not None:
        hidden = torch.arange(n, device=q.device)[None] > last[:, None]
    p = torch.softmax(s.masked_fill(hidden, -torch.inf), -1)
    o = torch.einsum("hqk,khd->qhd", p, v)
    A = torch.einsum("hqk,khd->qhd", p, v.abs())
    mag = torch.einsum("qhd,khd->hqk", q.abs(), k.abs()).masked_fill(hidden, 0).amax(-1).T[..., None] * abs(scale)
    d = mag * 1.4427 * 2.0 ** -17 + 2.0 ** -21
    tol = o.abs() * 2.0 ** -8 + A * (2.0 ** -11 + 2 * d) * 1.01 + n * 2.0 ** -33 * v.abs().amax() + 1e-30
    return o, tol


def _check_decode(out, q, k8, v8, table, lens, scale=D ** -0.5):
    for b, n in enumerate(lens):
        want, tol = _attention(q[b:b + 1], _row(k8, table[b], n), _row(v8, table[b], n), scale)
        err = (out[b:b + 1].double() - want).abs()
        assert (err <= tol).all(), f"request {b} of {n} keys: off by {(err / tol).max().item():.2f} of the tolerance"


# ---------------------------------------------------------------- append
def _append_case(T, nq, nkv, norm, seed, scale=1.0):
    ops = sub("ops")
    g = _gen(seed)
    qkv = (torch.randn(T, (nq + 2 * nkv) * D, device="cuda", generator=g) * scale).to(torch.bfloat16)
    pos = torch.randint(0, 4000, (T,), device="cuda", generator=g, dtype=torch.int32)
    cs = ops.rope_cos_sin(4096, D, 500000.0, "cuda")
    blocks = -(-T // PAGE) + 4
    slots = torch.randperm(blocks * PAGE, device="cuda", generator=g)[:T]
    kw = {}
    if norm:
        kw = dict(q_norm=(1 + 0.3 * torch.randn(D, device="cuda", generator=g)).to(torch.bfloat16),
                  k_norm=(1 + 0.3 * torch.randn(D, device="cuda", generator=g)).to(torch.bfloat16), eps=1e-6)
    return qkv, pos, cs, slots, blocks, kw


def _append_want(qkv, pos, cs, nq, nkv, kw):
    """fp64 q, k (rotated) and v, and the stored bytes of k and v."""
    ref, f8 = sub("ops.reference"), sub("ops.fp8_pages")
    T = qkv.shape[0]
    x = qkv.double().view(T, nq + 2 * nkv, D)
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]
    if kw:
        q, k = ref.rmsnorm(q, kw["q_norm"], kw["eps"]), ref.rmsnorm(k, kw["k_norm"], kw["eps"])
    q, k = ref.rope(q, pos, cs), ref.rope(k, pos, cs)
    return q, f8.quantize_rows(k), f8.quantize_rows(v)


def _check_append(q, k8, v8, qkv, pos, cs, slots, nq, nkv, kw):
    want_q, (kv, ke), (vv, ve) = _append_want(qkv, pos, cs, nq, nkv, kw)
    blk, off = slots // PAGE, slots % PAGE
    for pages, v, e in ((k8, kv, ke), (v8, vv, ve)):
        assert torch.equal(pages.exps[blk, :, off], e)
        assert torch.equal(_bytes_of(pages)[blk, :, off], v.view(torch.uint8))
    # q in fp32: two products and a sum, with the norm's 128-term sum, rsqrt and two products before it
    mag = want_q.abs() + want_q.roll(D // 2, -1).abs()
    tol = want_q.abs() * 2.0 ** -8 + mag * 2.0 ** -18
    assert ((q.double() - want_q).abs() <= tol * 1.01 + 1e-30).all()


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("T,nq,nkv", [(1, 32, 8), (1, 1, 1), (2, 4, 1), (17, 8, 1), (33, 6, 2), (64, 32, 8),
                                      (129, 64, 8), (1000, 8, 1), (515, 7, 7)])
def test_append_writes_the_definition(T, nq, nkv, norm):
    ops = sub("ops")
    qkv, pos, cs, slots, blocks, kw = _append_case(T, nq, nkv, norm, T)
    k8, v8 = ops.fp8_cache(blocks, nkv, "cuda")
    for p in (k8, v8):
        _bytes_of(p).fill_(0x55)
        p.exps.fill_(77)
    q = ops.rope_and_cache(qkv, pos, cs, nq, nkv, slots, k8, v8, **kw)
    _check_append(q, k8, v8, qkv, pos, cs, slots, nq, nkv, kw)
    # no other row changed
    rest = torch.ones(blocks * PAGE, dtype=torch.bool, device="cuda")
    rest[slots] = False
    for p in (k8, v8):
        assert (_bytes_of(p).transpose(1, 2).reshape(-1, nkv, D)[rest] == 0x55).all()
        assert (p.exps.transpose(1, 2).reshape(-1, nkv)[rest] == 77).all()


@pytest.mark.parametrize("scale", [0.0, 1e-38, 1e-30, 1e30])
def test_append_extreme_magnitudes(scale):
    ops = sub("ops")
    T, nq, nkv = 9, 4, 2
    qkv, pos, cs, slots, blocks, kw = _append_case(T, nq, nkv, False, 3, scale)
    k8, v8 = ops.fp8_cache(blocks, nkv, "cuda")
    ops.rope_and_cache(qkv, pos, cs, nq, nkv, slots, k8, v8)
    _, (kv, ke), (vv, ve) = _append_want(qkv, pos, cs, nq, nkv, kw)
    blk, off = slots // PAGE, slots % PAGE
    for pages, v, e in ((k8, kv, ke), (v8, vv, ve)):
        assert torch.equal(pages.exps[blk, :, off], e)
        assert torch.equal(_bytes_of(pages)[blk, :, off].view(torch.float8_e4m3fn).float(), v.float())


@pytest.mark.parametrize("case", ["edge", "beyond", "norm", "small"])
def test_append_rows_at_the_ends_of_the_range(case):
    """k rows that are finite in the definition but near or beyond fp32's
    largest number after the rotation or the norm, and rows whose elements reach
    below bf16's normal range."""
    ops = sub("ops")
    T, nq, nkv = 19, 4, 2
    qkv, pos, cs, slots, blocks, kw = _append_case(T, nq, nkv, case == "norm", 5, 1e-39 if case == "small" else 1.0)
    big = torch.finfo(torch.bfloat16).max
    if case == "edge":  # the rotation keeps a pair's length: these stay within (3.39e38, 3.41e38)
        qkv[:] = 0.0
        qkv.view(T, -1, D)[:, nq:, ::3] = big
    elif case == "beyond":
        qkv = torch.where(qkv < 0, -big, big).to(torch.bfloat16)
    elif case == "norm":
        kw["k_norm"] = torch.where(kw["k_norm"] > 1, big, -big / 4).to(torch.bfloat16)
        qkv.view(T, -1, D)[:, nq:, 5:] *= 0.01  # few dims carry the row: normalised elements up to sqrt(128 / 5)
    k8, v8 = ops.fp8_cache(blocks, nkv, "cuda")
    ops.rope_and_cache(qkv, pos, cs, nq, nkv, slots, k8, v8, **kw)
    _, (kv, ke), (vv, ve) = _append_want(qkv, pos, cs, nq, nkv, kw)
    blk, off = slots // PAGE, slots % PAGE
    for pages, v, e in ((k8, kv, ke), (v8, vv, ve)):
        assert not torch.isnan(v.float()).any()
        assert torch.equal(pages.exps[blk, :, off], e)
        assert torch.equal(_bytes_of(pages)[blk, :, off].view(torch.float8_e4m3fn).float(), v.float())
    assert (ke > 246).any() == (case != "small")


def test_append_borders_and_elements_that_are_not_finite():
    """Rows on and next to rounding borders (position 0: no rotation), and
    rows with NaN and infinities."""
    ops, f8 = sub("ops"), sub("ops.fp8_pages")
    nq, nkv, T = 1, 1, 6
    cs = ops.rope_cos_sin(4, D, 10000.0, "cuda")
    x = torch.zeros(T, 3, D, device="cuda")
    ties = torch.tensor([448.0, 17.0, 19.0, 21.0, -17.0, -19.0, 1.0625, 1.1875, 2.0 ** -10, 3 * 2.0 ** -10], device="cuda")
    x[0, 1:, :10] = ties
    x[1, 1:, :10] = -ties * 2.0 ** 5
    x[2, 1:] = 448.0
    x[3, 1:] = 450.0          # just past: the next exponent
    x[4, 1:] = torch.linspace(-2, 2, D, device="cuda")
    x[4, 1:, 3], x[4, 1:, 70] = float("nan"), float("inf")
    x[5, 1:] = float("-inf")
    qkv = x.reshape(T, -1).to(torch.bfloat16)
    pos = torch.zeros(T, dtype=torch.int32, device="cuda")
    slots = torch.arange(T, device="cuda") + 5
    k8, v8 = ops.fp8_cache(2, 1, "cuda")
    ops.rope_and_cache(qkv, pos, cs, nq, nkv, slots, k8, v8)
    v, e = f8.quantize_rows(qkv.view(T, 3, D)[:, 2:].float())
    got = _bytes_of(v8)[slots // PAGE, :, slots % PAGE].view(torch.float8_e4m3fn).float()
    assert torch.equal(v8.exps[slots // PAGE, :, slots % PAGE], e)
    assert torch.equal(got.nan_to_num(nan=1e9), v.float().nan_to_num(nan=1e9))
    # k: cos 1, sin 0 keeps finite rows; 0 * inf makes the partner NaN as well
    assert torch.equal(k8.exps[slots // PAGE, :, slots % PAGE][:4], e[:4])
    gk = _bytes_of(k8)[slots // PAGE, :, slots % PAGE].view(torch.float8_e4m3fn).float()
    assert torch.equal(gk[:4], v.float()[:4])
    assert torch.isnan(gk[4, 0, [3, 6, 67, 70]]).all() and torch.isnan(gk[4]).sum() == 4
    assert torch.isnan(gk[5]).all()


@pytest.mark.parametrize("T", [5, 300])
def test_append_skips_slots_outside_and_keeps_the_last_of_equal_ones(T):
    ops = sub("ops")
    nq, nkv = 4, 2
    qkv, pos, cs, slots, blocks, kw = _append_case(T, nq, nkv, False, 9)
    slots[1] = -1
    slots[2] = blocks * PAGE
    slots[0] = slots[T - 1]           # the last token keeps it
    if T > 100:
        slots[40:90:7] = slots[97]    # several tokens, one slot; 97 is the last
    k8, v8 = ops.fp8_cache(blocks, nkv, "cuda")
    k0, v0 = k8.values.view(torch.uint8).clone(), v8.exps.clone()
    q = ops.rope_and_cache(qkv, pos, cs, nq, nkv, slots, k8, v8)
    last = {int(s): t for t, s in enumerate(slots.tolist()) if 0 <= s < blocks * PAGE}
    keep = torch.tensor(sorted(last.values()), device="cuda")
    want_q, (kv, ke), (vv, ve) = _append_want(qkv, pos, cs, nq, nkv, kw)
    blk, off = slots[keep] // PAGE, slots[keep] % PAGE
    for pages, v, e in ((k8, kv, ke), (v8, vv, ve)):
        assert torch.equal(_bytes_of(pages)[blk, :, off], v.view(torch.uint8)[keep])
        assert torch.equal(pages.exps[blk, :, off], e[keep])
        mask = torch.ones(blocks, PAGE, dtype=torch.bool, device="cuda")
        mask[blk, off] = False
        assert (_bytes_of(pages).transpose(1, 2)[mask] == 0).all()
    assert ((q.double() - want_q).abs() <= want_q.abs() * 2.0 ** -8 + 2e-5).all()


def test_append_positions_outside_the_table_take_its_ends():
    ops = sub("ops")
    nq, nkv, T = 4, 2, 4
    qkv, pos, cs, slots, blocks, kw = _append_case(T, nq, nkv, False, 2)
    cs = cs[:100].contiguous()
    bad = torch.tensor([-5, 100, 2 ** 31 - 1, 50], dtype=torch.int32, device="cuda")
    k8, v8 = ops.fp8_cache(blocks, nkv, "cuda")
    q = ops.rope_and_cache(qkv, bad, cs, nq, nkv, slots, k8, v8)
    _check_append(q, k8, v8, qkv, bad.clamp(0, 99), cs, slots, nq, nkv, kw)


def test_append_nothing():
    ops = sub("ops")
    k8, v8 = ops.fp8_cache(1, 1, "cuda")
    cs = ops.rope_cos_sin(4, D, 10000.0, "cuda")
    q = ops.rope_and_cache(torch.zeros(0, 3 * D, device="cuda", dtype=torch.bfloat16),
                           torch.zeros(0, device="cuda", dtype=torch.int32), cs, 1, 1,
                           torch.zeros(0, device="cuda", dtype=torch.int64), k8, v8)
    assert q.shape == (0, 1, D)


# ---------------------------------------------------------------- read
@pytest.mark.parametrize("lens,nkv", [([1], 1), ([16], 2), ([17, 0, 31, 32, 33], 3), ([777], 8),
                                      ([5, 300, 0, 64, 1029, 1], 8)])
def test_read_pages(lens, nkv):
    ops = sub("ops")
    k8, v8, kvl, table = _cache(lens, nkv, seed=len(lens), spread=30)
    R, cols = table.shape
    fresh = ops.read_pages(k8, v8, table, kvl)
    given = [torch.full((R * cols + 2, nkv, PAGE, D), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ops.read_pages(k8, v8, table, kvl, k_out=given[0], v_out=given[1])
    for pages, a, b in ((k8, fresh[0], given[0]), (v8, fresh[1], given[1])):
        for r, n in enumerate(lens):
            used = -(-n // PAGE)
            for out, rest in ((a, 0.0), (b, 7.0)):
                mine = out[r * cols:(r + 1) * cols]
                rows = mine.transpose(1, 2).reshape(-1, nkv, D)
                assert torch.equal(rows[:n].double(), _row(pages, table[r], n))
                assert (rows[n:used * PAGE] == 0).all() and (rows[used * PAGE:] == rest).all()
        assert (b[R * cols:] == 7.0).all()


def test_read_pages_by_plan_strided_tables_and_bad_pages():
    ops = sub("ops")
    lens, nkv = [40, 0, 7, 100], 2
    k8, v8, kvl, table = _cache(lens, nkv, seed=4, columns=7)
    wide = torch.full((4, 12), 10 ** 9, dtype=torch.int32, device="cuda")
    wide[:, 2:9] = table
    view = wide[:, 2:9]
    plan = ops.page_plan(lens, 7)
    out = [torch.zeros(plan.pages, nkv, PAGE, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ops.read_pages(k8, v8, view, kvl, out_table=plan.table.cuda(), k_out=out[0], v_out=out[1])
    dense = ops.read_pages(k8, v8, table, kvl)
    at = 0
    for r, n in enumerate(lens):
        for i in range(-(-n // PAGE)):
            assert torch.equal(out[0][at], dense[0][r * 7 + i]) and torch.equal(out[1][at], dense[1][r * 7 + i])
            at += 1
    # blocks outside the cache read as zeros; output entries outside the output are skipped
    bad = table.clone()
    bad[0, 1], bad[3, 0] = -7, k8.shape[0]
    t = plan.table.cuda()
    t[2, 0], t[3, 1] = plan.pages, -3
    out = [torch.full((plan.pages, nkv, PAGE, D), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    ops.read_pages(k8, v8, bad, kvl, out_table=t, k_out=out[0], v_out=out[1])
    assert (out[0][1] == 0).all() and (out[1][4] == 0).all()                # request 0 page 1, request 3 page 0
    assert (out[0][3] == 3.0).all() and (out[1][5] == 3.0).all()            # the skipped ones
    assert torch.equal(out[0][0], dense[0][0]) and torch.equal(out[1][6], dense[1][3 * 7 + 2])
    # a length past the table reads the table's pages only
    over = torch.full_like(kvl, 10 ** 6)
    k, _ = ops.read_pages(k8, v8, table[3:], over[3:])
    assert torch.equal(k[:6, :, :4], dense[0][21:27, :, :4])
    # nothing to read
    assert ops.read_pages(k8, v8, table[:0], kvl[:0])[0].shape[0] == 0
    assert ops.read_pages(k8, v8, table[:, :0], kvl)[0].shape[0] == 0


def test_read_pages_of_every_exponent_and_number():
    ops = sub("ops")
    cache = ops.fp8_cache(32, 1, "cuda")
    for i, c in enumerate(cache):
        _bytes_of(c).view(-1, D)[:] = (torch.arange(D, device="cuda") + 128 * i).to(torch.uint8)
        c.exps[:, 0] = torch.arange(1, 513, device="cuda").remainder(254).add(1).to(torch.uint8).view(32, PAGE)
    table = torch.arange(32, dtype=torch.int32, device="cuda")[None]
    got = ops.read_pages(*cache, table, torch.tensor([512], dtype=torch.int32, device="cuda"))
    for c, x in zip(cache, got):
        want = torch.nan_to_num(c.dequantize().float(), nan=7.0)
        assert torch.equal(torch.nan_to_num(x.float(), nan=7.0), want) and want.isfinite().any()


# ---------------------------------------------------------------- decode
LENS = [1, 0, 2, 15, 16, 17, 31, 33, 100, 500, 777, 2049]


@pytest.mark.parametrize("nq,nkv", [(1, 1), (3, 1), (4, 1), (7, 1), (8, 1), (9, 1), (16, 1), (32, 8), (64, 8),
                                    (6, 2), (48, 3)])
def test_decode_heads_and_lengths(nq, nkv):
    ops = sub("ops")
    k8, v8, kvl, table = _cache(LENS, nkv, seed=nq)
    q = torch.randn(len(LENS), nq, D, device="cuda", generator=_gen(nq)).to(torch.bfloat16)
    out = ops.decode_attention(q, k8, v8, kvl, table)
    _check_decode(out, q, k8, v8, table, LENS)
    assert (out[1] == 0).all()
    # call after call the same bits, whatever the other requests' lengths
    for _ in range(3):
        assert torch.equal(ops.decode_attention(q, k8, v8, kvl, table), out)


@pytest.mark.parametrize("lens", [[1], [16], [4096], [9000], [4096, 3], [33000, 0, 1, 20000]])
def test_decode_few_long_requests(lens):
    ops = sub("ops")
    for nq, nkv in ((32, 8), (8, 1), (16, 1)):
        k8, v8, kvl, table = _cache(lens, nkv, seed=lens[0])
        q = torch.randn(len(lens), nq, D, device="cuda", generator=_gen(1)).to(torch.bfloat16)
        out = ops.decode_attention(q, k8, v8, kvl, table)
        _check_decode(out, q, k8, v8, table, lens)


@pytest.mark.parametrize("B,nq,nkv", [(70, 8, 2), (300, 4, 4), (1100, 2, 1)])
def test_decode_many_requests(B, nq, nkv):
    ops = sub("ops")
    lens = [(r * 37) % 130 for r in range(B)]
    k8, v8, kvl, table = _cache(lens, nkv, seed=B)
    q = torch.randn(B, nq, D, device="cuda", generator=_gen(2)).to(torch.bfloat16)
    out = ops.decode_attention(q, k8, v8, kvl, table)
    _check_decode(out, q, k8, v8, table, lens)


@pytest.mark.parametrize("spread,qscale,scale", [(12, 1.0, None), (0, 30.0, None), (0, 1e-20, 1e20), (0, 1e20, 1e-20),
                                                 (6, 1.0, -0.3), (0, 1.0, 0.0), (40, 1.0, 1e-9)])
def test_decode_magnitudes(spread, qscale, scale):
    """Rows whose scales differ by up to 2^80, sharp and flat softmaxes, the
    weight of one row against many, negative and zero scales."""
    ops = sub("ops")
    lens, nq, nkv = [1, 40, 700, 3000], 16, 2
    k8, v8, kvl, table = _cache(lens, nkv, seed=17, spread=spread)
    if spread:  # k rows of one magnitude, so that the softmax is not one key's
        k8 = _cache(lens, nkv, seed=17)[0]
    q = (torch.randn(4, nq, D, device="cuda", generator=_gen(3)) * qscale).to(torch.bfloat16)
    out = ops.decode_attention(q, k8, v8, kvl, table, scale=scale)
    _check_decode(out, q, k8, v8, table, lens, scale if scale is not None else D ** -0.5)


@pytest.mark.parametrize("byte", [1, 5, 9, 10, 254 - 8])
def test_decode_extreme_value_exponents(byte):
    """Value exponents at the ends of what Fp8Pages holds. The tolerance is
    _attention's without its absolute part; bf16's smallest step is 2^-133."""
    ops = sub("ops")
    lens = [7, 40, 3000]
    k8, v8, kvl, table = _cache(lens, 2, seed=byte)
    v8.exps.copy_(torch.where(v8.exps == 255, v8.exps, torch.full_like(v8.exps, byte)))
    q = torch.randn(3, 8, D, device="cuda", generator=_gen(byte)).to(torch.bfloat16)
    out = ops.decode_attention(q, k8, v8, kvl, table)
    for b, n in enumerate(lens):
        v = sub("ops.fp8_pages").dequantize_rows(*_live_rows(v8, table[b], n)).double()
        want, tol = _attention(q[b:b + 1], _row(k8, table[b], n), v, D ** -0.5)
        assert ((out[b:b + 1].double() - want).abs() <= tol - 1e-30 + 2.0 ** -133).all(), (byte, n)


def _spread_tol(p, v, n):
    """What the weights' f16 grid may cost a row of probabilities p [nq, n] over
    v [n, nq, 128]: the key that contributes most has a weight of 2^10 at least,
    the others are off by half of f16's smallest step, 2^-25, times their
    e4m3 number, of which a row's largest is in (224, 448]."""
    top = v.abs().amax(-1).T  # [nq, n]
    return n * 2.0 ** -34 * (p * top).amax(-1, keepdim=True)


@pytest.mark.parametrize("nq,nkv", [(8, 2), (16, 1), (3, 1)])
@pytest.mark.parametrize("gap", [20, 24, 28, 31, 33, 40, 60, 100])
@pytest.mark.parametrize("n", [40, 3000])
def test_decode_loud_value_rows_that_no_head_attends_to(n, gap, nq, nkv):
    """Rows of value 2^gap times the others' whose weight is 2^-(gap + 40) of
    theirs at most: they count for nothing, the quiet ones for all. Loud rows
    come first, last and in between."""
    _check_loud(n, nq, nkv, gap, -30, gap + 60.0)


@pytest.mark.parametrize("nq,nkv", [(8, 2), (16, 1)])
@pytest.mark.parametrize("n", [40, 3000])
def test_decode_weights_below_fp32_count_as_zero(n, nq, nkv):
    """Rows 2^200 times the others, of a weight (2^-150) that fp32 does not have."""
    _check_loud(n, nq, nkv, 200, -100, 160.0, counted=False)


def _check_loud(n, nq, nkv, gap, low, away, counted=True):
    """Loud rows of value 2^(low + gap) among quiet ones of 2^low, their scores
    0.7 away ln-units lower."""
    ops, f8 = sub("ops"), sub("ops.fp8_pages")
    k8, v8, kvl, table = _cache([n], nkv, seed=gap)
    g = _gen(gap + n)
    loud = torch.zeros(table.shape[1] * PAGE, dtype=torch.bool, device="cuda")
    loud[[0, 1, n // 2, n - 1]] = True
    x = torch.randn(loud.numel(), nkv, D, device="cuda", generator=g)
    v = torch.where(loud[:, None, None], x * 2.0 ** (low + gap), x * 2.0 ** low)
    k = 0.1 * torch.randn(loud.numel(), nkv, D, device="cuda", generator=g)
    k[..., 0] = torch.where(loud, -away, 0.0)[:, None]
    for pages, rows in ((k8, k), (v8, v)):
        values, exps = f8.quantize_rows(rows.view(-1, PAGE, nkv, D).transpose(1, 2))
        _bytes_of(pages)[table[0].long()] = values.view(torch.uint8)
        pages.exps[table[0].long()] = exps
    q = torch.randn(1, nq, D, device="cuda", generator=g).to(torch.bfloat16)
    q[..., 0] = 0.7
    out = ops.decode_attention(q, k8, v8, kvl, table, scale=1.0).double()
    G = nq // nkv
    kk, vv = (_row(c, table[0], n).repeat_interleave(G, 1) for c in (k8, v8))
    p = torch.softmax(torch.einsum("hd,khd->hk", q[0].double(), kk), -1)
    if not counted:
        p = torch.where(loud[:n], 0.0, p)
    want = torch.einsum("hk,khd->hd", p, vv)
    # _attention's bound with _spread_tol in the place of its absolute part
    A = torch.einsum("hk,khd->hd", p, vv.abs())
    mag = torch.einsum("hd,khd->hk", q[0].double().abs(), kk.abs()).amax(-1, keepdim=True)
    tol = want.abs() * 2.0 ** -8 + A * (2.0 ** -11 + 2 * (mag * 1.4427 * 2.0 ** -17 + 2.0 ** -21)) * 1.01
    tol = tol + _spread_tol(p, vv, n)
    err = (out[0] - want).abs()
    assert (err <= tol).all(), f"off by {(err / tol).max().item():.2f} of the tolerance"


def _live_rows(pages, table_row, n):
    """(values [n, nkv, 128], exps [n, nkv]) of a request."""
    blocks = table_row[:-(-n // PAGE)].long()
    values = _bytes_of(pages)[blocks].transpose(1, 2).flatten(0, 1)[:n]
    return values.view(torch.float8_e4m3fn), pages.exps[blocks].transpose(1, 2).flatten(0, 1)[:n]


def test_decode_long_sums_of_the_smallest_values():
    """Rows of one value at the smallest exponent, equal weights: the mean is
    that value, however long the row (2^-117 over 130056 keys leaves fp32's
    normal range on the way)."""
    ops = sub("ops")
    n, B = 130056, 1200
    k8, v8 = ops.fp8_cache(1, 1, "cuda")
    _bytes_of(v8).fill_(0x3E)  # 1.75
    v8.exps.fill_(10)
    table = torch.zeros(1, -(-n // PAGE), dtype=torch.int32, device="cuda").expand(B, -1)
    kvl = torch.full((B,), n, dtype=torch.int32, device="cuda")
    q = torch.zeros(B, 1, D, dtype=torch.bfloat16, device="cuda")
    out = ops.decode_attention(q, k8, v8, kvl, table).double()
    # a rounding to bf16 of a value next to 1.75, weights and sums in fp32
    assert ((out * 2.0 ** 117 - 1.75).abs() <= 2.0 ** -8 + 1.75 * 2.0 ** -11).all()


def test_decode_scores_that_rise_along_the_cache():
    """The running maximum moves on every page; an early key of weight zero."""
    ops, f8 = sub("ops"), sub("ops.fp8_pages")
    n, nkv, nq = 1500, 1, 8
    k8, v8, kvl, table = _cache([n], nkv, seed=5)
    x = torch.zeros(-(-n // PAGE) * PAGE, nkv, D, device="cuda")
    x[:, 0, 0] = torch.arange(x.shape[0], device="cuda") * 0.25
    x[:, 0, 1:] = 0.1 * torch.randn(x.shape[0], D - 1, device="cuda", generator=_gen(5))
    v, e = f8.quantize_rows(x.view(-1, PAGE, nkv, D).transpose(1, 2))
    _bytes_of(k8)[table[0].long()] = v.view(torch.uint8)
    k8.exps[table[0].long()] = e
    for sign in (1.0, -1.0):
        q = torch.randn(1, nq, D, device="cuda", generator=_gen(6)).to(torch.bfloat16)
        q[..., 0] = 8.0 * sign
        out = ops.decode_attention(q, k8, v8, kvl, table)
        _check_decode(out, q, k8, v8, table, [n])


def test_decode_non_finite_inputs_stay_in_their_rows():
    ops = sub("ops")
    lens, nq, nkv = [50, 50, 50, 600], 8, 2
    k8, v8, kvl, table = _cache(lens, nkv, seed=8)
    q = torch.randn(4, nq, D, device="cuda", generator=_gen(8)).to(torch.bfloat16)
    exact = [_attention(q[b:b + 1], _row(k8, table[b], n), _row(v8, table[b], n), D ** -0.5)
             for b, n in enumerate(lens)]
    want, tol = (torch.cat(x) for x in zip(*exact))
    q[0, 1, 5] = float("nan")
    q[1, 2, 9] = float("inf")
    _bytes_of(v8)[table[2, 1].long(), 1, 3, 7] = 0x7F    # one element of one row: heads 4..7, dim 7
    _bytes_of(k8)[table[3, 20].long(), 0, 2, 0] = 0x7F   # one key: heads 0..3
    out = ops.decode_attention(q, k8, v8, kvl, table)
    bad = torch.zeros(4, nq, D, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[1, 2] = True
    bad[2, 4:, 7] = True
    bad[3, :4] = True
    assert torch.isnan(out[bad]).all()
    # The others: the definition's values. Not the same bits as without the
    # NaN, since the heads that share a kv head move their running maxima
    # together, and the weights' rounding goes with them.
    assert ((out.double() - want).abs() <= tol)[~bad].all()


def test_decode_tables_lengths_and_pages_outside():
    ops = sub("ops")
    lens, nq, nkv = [100, 40, 33], 8, 2
    k8, v8, kvl, table = _cache(lens, nkv, seed=11, columns=8)
    q = torch.randn(3, nq, D, device="cuda", generator=_gen(4)).to(torch.bfloat16)
    out = ops.decode_attention(q, k8, v8, kvl, table)
    wide = torch.full((3, 20), 10 ** 9, dtype=torch.int32, device="cuda")
    wide[:, 5:13] = table
    assert torch.equal(ops.decode_attention(q, k8, v8, kvl, wide[:, 5:13]), out)
    # lengths behind the table end at it; negative ones are empty
    over = torch.tensor([10 ** 9, 40, -5], dtype=torch.int32, device="cuda")
    full = table[:, :6]
    got = ops.decode_attention(q, k8, v8, over, full)
    _check_decode(got[:2], q[:2], k8, v8, full, [96, 40])
    assert (got[2] == 0).all()
    # blocks outside the cache: their keys do not count
    bad = table.clone()
    bad[0, 2], bad[1, 0], bad[1, 1], bad[1, 2] = -1, k8.shape[0], 2 ** 31 - 1, -2 ** 31
    got = ops.decode_attention(q, k8, v8, kvl, bad)
    k = torch.cat([_row(k8, table[0], 100)[:32], _row(k8, table[0], 100)[48:]])
    v = torch.cat([_row(v8, table[0], 100)[:32], _row(v8, table[0], 100)[48:]])
    want, tol = _attention(q[:1], k, v, D ** -0.5)
    assert ((got[:1].double() - want).abs() <= tol).all()
    assert (got[1] == 0).all() and torch.equal(got[2], out[2])
    # no requests, no columns
    assert ops.decode_attention(q[:0], k8, v8, kvl[:0], table[:0]).shape == (0, nq, D)
    assert (ops.decode_attention(q, k8, v8, kvl, table[:, :0]) == 0).all()
    # rows of an output given are all that is written
    o = torch.full((5, nq, D), 9.0, dtype=torch.bfloat16, device="cuda")
    assert ops.decode_attention(q, k8, v8, kvl, table, out=o[1:4]).data_ptr() == o[1].data_ptr()
    assert torch.equal(o[1:4], out) and (o[0] == 9).all() and (o[4] == 9).all()


def test_decode_shared_pages():
    """Two requests that share a prefix's pages, and one page named twice."""
    ops = sub("ops")
    k8, v8, kvl, table = _cache([80, 80], 2, seed=13)
    table[1, :3] = table[0, :3]
    table[1, 4] = table[1, 3]
    q = torch.randn(2, 8, D, device="cuda", generator=_gen(4)).to(torch.bfloat16)
    out = ops.decode_attention(q, k8, v8, kvl, table)
    _check_decode(out, q, k8, v8, table, [80, 80])


def test_decode_far_offsets():
    """Pages whose bytes lie past 2^31 and 2^32 of the cache's start."""
    ops = sub("ops")
    nkv, nq, n = 8, 32, 200
    k8, v8, kvl, table = _cache([n], nkv, seed=21)
    blocks = (5 << 30) // (nkv * PAGE * D)
    big = [ops.Fp8Pages(torch.empty(blocks, nkv, PAGE, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
                        torch.empty(blocks, nkv, PAGE, dtype=torch.uint8, device="cuda")) for _ in range(2)]
    far = torch.linspace(3, blocks - 1, table.shape[1], device="cuda").long().flip(0)
    for a, b in zip(big, (k8, v8)):
        _bytes_of(a)[far] = _bytes_of(b)[table[0].long()]
        a.exps[far] = b.exps[table[0].long()]
    q = torch.randn(1, nq, D, device="cuda", generator=_gen(4)).to(torch.bfloat16)
    t = far.to(torch.int32)[None]
    out = ops.decode_attention(q, *big, kvl, t)
    assert torch.equal(out, ops.decode_attention(q, k8, v8, kvl, table))
    k, v = ops.read_pages(*big, t, kvl)
    want = ops.read_pages(k8, v8, table, kvl)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    # a row written at the far end
    cs = ops.rope_cos_sin(8, D, 10000.0, "cuda")
    qkv = torch.randn(1, (nq + 2 * nkv) * D, device="cuda", generator=_gen(1)).to(torch.bfloat16)
    pos = torch.tensor([3], dtype=torch.int32, device="cuda")
    slot = torch.tensor([blocks * PAGE - 2], device="cuda")
    ops.rope_and_cache(qkv, pos, cs, nq, nkv, slot, *big)
    _, (kb, ke), (vb, ve) = _append_want(qkv, pos, cs, nq, nkv, {})
    assert torch.equal(_bytes_of(big[0])[-1, :, -2], kb[0].view(torch.uint8))
    assert torch.equal(_bytes_of(big[1])[-1, :, -2], vb[0].view(torch.uint8)) and torch.equal(big[1].exps[-1, :, -2], ve[0])


def test_separate_exponent_tensors():
    """Exponents in tensors of their own, and with padding between heads."""
    ops = sub("ops")
    k8, v8, kvl, table = _cache([70, 5], 2, seed=2)
    q = torch.randn(2, 4, D, device="cuda", generator=_gen(4)).to(torch.bfloat16)
    out = ops.decode_attention(q, k8, v8, kvl, table)
    pad = torch.empty(k8.shape[0], 2, 48, dtype=torch.uint8, device="cuda")
    pad[..., 16:32] = k8.exps
    a, b = ops.Fp8Pages(k8.values, pad[..., 16:32]), ops.Fp8Pages(v8.values, v8.exps.contiguous())
    assert torch.equal(ops.decode_attention(q, a, b, kvl, table), out)
    assert torch.equal(ops.read_pages(a, b, table, kvl)[0], ops.read_pages(k8, v8, table, kvl)[0])


# ---------------------------------------------------------------- prefill
def _check_prefill(out, q, k8, v8, table, q_lens, kv_lens):
    """The tcgen05 kernel rounds its weights (at most 2^8) to bf16: ub A
    instead of u16 A; the keys and values it reads are the cache's exactly."""
    row = 0
    for r, (ql, n) in enumerate(zip(q_lens, kv_lens)):
        last = torch.arange(n - ql, n, device="cuda")
        k, v = _row(k8, table[r], n), _row(v8, table[r], n)
        want, tol = _attention(q[row:row + ql], k, v, D ** -0.5, last)
        A, _ = _attention(q[row:row + ql], k, v.abs(), D ** -0.5, last)
        err = (out[row:row + ql].double() - want).abs()
        assert (err <= tol + A * 2.0 ** -8 * 1.01).all(), f"request {r}: {(err / (tol + A * 2.0 ** -8)).max().item()}"
        row += ql


@pytest.mark.parametrize("nq,nkv", [(32, 8), (8, 1), (3, 1)])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("planned", [False, True])
def test_prefill_over_the_cache(nq, nkv, splits, planned):
    ops = sub("ops")
    kv_lens, q_lens = [100, 264, 1, 777, 16], [100, 64, 1, 257, 3]
    k8, v8, kvl, table = _cache(kv_lens, nkv, seed=nq)
    q = torch.randn(sum(q_lens), nq, D, device="cuda", generator=_gen(1)).to(torch.bfloat16)
    cu = torch.tensor([0] + q_lens, device="cuda").cumsum(0).to(torch.int32)
    plan = ops.page_plan(kv_lens, table.shape[1]) if planned else None
    if planned:
        plan.table = plan.table.cuda()
    out = ops.prefill_attention(q, k8, v8, cu, kvl, table, ops.prefill_tiles(q_lens).cuda(), splits=splits, plan=plan)
    torch.cuda.synchronize()
    assert ops.gemm_error() == 0
    _check_prefill(out, q, k8, v8, table, q_lens, kv_lens)


def _prefill(ops, q, k8, v8, q_lens, kvl, table, **kw):
    cu = torch.tensor([0] + q_lens, device="cuda").cumsum(0).to(torch.int32)
    return ops.prefill_attention(q, k8, v8, cu, kvl, table, ops.prefill_tiles(q_lens).cuda(), **kw)


@pytest.mark.parametrize("kv_lens,q_lens", [([63], [63]), ([64], [1]), ([65], [65]), ([129], [2]), ([1], [1]),
                                            ([2000, 256, 511], [600, 256, 255]), ([1027], [515]),
                                            ([300, 17, 129, 640], [257, 17, 128, 1])])
def test_prefill_tile_borders(kv_lens, q_lens):
    ops = sub("ops")
    nq, nkv = 4, 2
    k8, v8, kvl, table = _cache(kv_lens, nkv, seed=kv_lens[0], spread=3)
    q = torch.randn(sum(q_lens), nq, D, device="cuda", generator=_gen(2)).to(torch.bfloat16)
    out = _prefill(ops, q, k8, v8, q_lens, kvl, table)
    _check_prefill(out, q, k8, v8, table, q_lens, kv_lens)
    assert ops.gemm_error() == 0


def test_prefill_rows_without_keys_and_neighbours_with_nan():
    """A request without cached keys gives zeros; NaN rows of one request stay
    in it, although its pages lie next to the others' in the scratch."""
    ops = sub("ops")
    kv_lens, q_lens, nq, nkv = [70, 0, 30, 100], [20, 9, 30, 5], 4, 2
    k8, v8, kvl, table = _cache(kv_lens, nkv, seed=3)
    q = torch.randn(sum(q_lens), nq, D, device="cuda", generator=_gen(2)).to(torch.bfloat16)
    for splits in (1, 2):
        out = _prefill(ops, q, k8, v8, q_lens, kvl, table, splits=splits)
        assert (out[20:29] == 0).all()
        for r, a, b in ((0, 0, 20), (2, 29, 59), (3, 59, 64)):
            _check_prefill(out[a:b], q[a:b], k8, v8, table[r:r + 1], [b - a], kv_lens[r:r + 1])
    good = _prefill(ops, q, k8, v8, q_lens, kvl, table)
    _bytes_of(v8)[table[2, 0].long()] = 0x7F
    bad = _prefill(ops, q, k8, v8, q_lens, kvl, table)
    assert torch.isnan(bad[29:59]).all()
    assert torch.equal(bad[:29], good[:29]) and torch.equal(bad[59:], good[59:])
    # nothing to attend with, and no columns at all
    assert _prefill(ops, q[:0], k8, v8, [], kvl[:0], table[:0]).shape == (0, nq, D)
    assert (_prefill(ops, q[:5], k8, v8, [5], kvl[:1], table[:1, :0]) == 0).all()
    with pytest.raises(RuntimeError, match="positive scale"):
        _prefill(ops, q, k8, v8, q_lens, kvl, table, scale=0.0)


@pytest.mark.parametrize("splits", [1, 2])
def test_prefill_by_plans_in_any_order(splits):
    """Plans that scatter a request's pages, leave room between them, serve
    longer lengths, or run backwards: the same bits as the packed one."""
    ops = sub("ops")
    kv_lens, q_lens, nq, nkv = [333, 70, 1029, 64], [100, 70, 300, 1], 4, 2
    k8, v8, kvl, table = _cache(kv_lens, nkv, seed=6, columns=70)
    q = torch.randn(sum(q_lens), nq, D, device="cuda", generator=_gen(2)).to(torch.bfloat16)
    packed = ops.page_plan(kv_lens, 70)
    want = _prefill(ops, q, k8, v8, q_lens, kvl, table, splits=splits, plan=ops.PagePlan(packed.table.cuda(), packed.pages))
    _check_prefill(want, q, k8, v8, table, q_lens, kv_lens)
    n = packed.pages
    perm = torch.randperm(n, generator=torch.Generator().manual_seed(0)).to(torch.int32)
    backwards = torch.arange(n - 1, -1, -1, dtype=torch.int32)
    room = 3 * torch.arange(n, dtype=torch.int32)
    for order, pages in ((perm, n), (backwards, n), (room, 3 * n)):
        t = torch.where(packed.table >= 0, order[packed.table.clamp_min(0).long()], packed.table)
        got = _prefill(ops, q, k8, v8, q_lens, kvl, table, splits=splits, plan=ops.PagePlan(t.cuda(), pages))
        assert torch.equal(got, want)
    longer = ops.page_plan([n + 100 for n in kv_lens], 70)
    got = _prefill(ops, q, k8, v8, q_lens, kvl, table, splits=splits, plan=ops.PagePlan(longer.table.cuda(), longer.pages))
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    assert ops.gemm_error() == 0


def test_prefill_by_a_plan_that_lacks_pages():
    """Pages that the plan does not place count as zeros, and the error word
    says so; the requests that it places are right."""
    ops = sub("ops")
    kv_lens, q_lens, nq, nkv = [333, 70, 200], [33, 70, 5], 4, 2
    k8, v8, kvl, table = _cache(kv_lens, nkv, seed=6)
    q = torch.randn(sum(q_lens), nq, D, device="cuda", generator=_gen(2)).to(torch.bfloat16)
    short = ops.page_plan([160, 70, 200], table.shape[1])
    t = short.table.cuda()
    t[2, 1], t[2, 5] = short.pages, -2 ** 31
    err = ops.workspace("cuda").err
    try:
        out = _prefill(ops, q, k8, v8, q_lens, kvl, table, plan=ops.PagePlan(t, short.pages))
        none = _prefill(ops, q, k8, v8, q_lens, kvl, table, plan=ops.PagePlan(torch.full_like(t, -1), 0))
        torch.cuda.synchronize()
        assert ops.gemm_error() == 24
    finally:
        err.zero_()
    _check_prefill(out[33:103], q[33:103], k8, v8, table[1:2], [70], [70])
    for r, a, b, lost in ((0, 0, 33, slice(160, 333)), (2, 103, 108, [*range(16, 32), *range(80, 96)])):
        n = kv_lens[r]
        k, v = _row(k8, table[r], n).clone(), _row(v8, table[r], n).clone()
        k[lost], v[lost] = 0.0, 0.0
        last = torch.arange(n - (b - a), n, device="cuda")
        want, tol = _attention(q[a:b], k, v, D ** -0.5, last)
        A, _ = _attention(q[a:b], k, v.abs(), D ** -0.5, last)
        assert ((out[a:b].double() - want).abs() <= tol + A * 2.0 ** -8 * 1.01).all()
    assert (none == 0).all()


@pytest.mark.parametrize("seed", range(10))
def test_decode_drawn_batches(seed):
    """Batches of mixed lengths, so that runs of the work list begin and end
    anywhere in pairs, pages and the room behind them."""
    import random

    ops = sub("ops")
    rng = random.Random(seed)
    nkv = rng.choice((1, 2, 3, 8))
    nq = nkv * rng.choice((1, 2, 5, 8, 11, 16))
    B = rng.choice((1, 2, 7, 40, 150, 333))
    top = rng.choice((40, 200, 900, 6000)) if B < 100 else rng.choice((40, 200, 700))
    lens = [0 if rng.random() < 0.1 else rng.choice((rng.randint(1, 30), rng.randint(1, top))) for _ in range(B)]
    k8, v8, kvl, table = _cache(lens, nkv, seed=seed, columns=-(-max(max(lens), 1) // PAGE) + rng.randint(0, 3))
    q = torch.randn(B, nq, D, device="cuda", generator=_gen(seed)).to(torch.bfloat16)
    out = ops.decode_attention(q, k8, v8, kvl, table)
    _check_decode(out, q, k8, v8, table, lens)


def test_decode_among_other_requests():
    """A request among others of changing lengths: the runs' borders move, and
    with them the last bits; each result is within the tolerance, and the same
    batch gives the same bits again."""
    ops = sub("ops")
    nq, nkv, n = 8, 2, 777
    k8, v8, _, table = _cache([n] + [3000] * 15, nkv, seed=1)
    q = torch.randn(16, nq, D, device="cuda", generator=_gen(1)).to(torch.bfloat16)
    want, tol = _attention(q[:1], _row(k8, table[0], n), _row(v8, table[0], n), D ** -0.5)
    for others in ([3000] * 15, [0] * 15, [1] * 15, [100, 2000] * 7 + [5], list(range(0, 3000, 200))):
        kvl = torch.tensor([n] + others, dtype=torch.int32, device="cuda")
        out = ops.decode_attention(q, k8, v8, kvl, table)
        assert ((out[:1].double() - want).abs() <= tol).all()
        assert torch.equal(ops.decode_attention(q, k8, v8, kvl, table), out)


# ---------------------------------------------------------------- together
def test_append_then_attend():
    """A prompt in two chunks, then tokens one by one, as a model's layer
    makes the calls; every attention against the definition."""
    ops = sub("ops")
    nq, nkv = 8, 2
    k8, v8 = ops.fp8_cache(40, nkv, "cuda")
    for p in (k8, v8):
        _bytes_of(p).fill_(0x7F)
        p.exps.fill_(255)
    table = torch.randperm(40, device="cuda", generator=_gen(0))[:20].to(torch.int32).view(2, 10)
    cs = ops.rope_cos_sin(256, D, 500000.0, "cuda")
    lens = [0, 0]
    for step, new in enumerate([[70, 33], [31, 64], [1, 1], [1, 1], [1, 1]]):
        T = sum(new)
        pos = torch.cat([torch.arange(a, a + b, device="cuda") for a, b in zip(lens, new)])
        row = torch.tensor([0] * new[0] + [1] * new[1], device="cuda")
        slots = table.long()[row, pos // PAGE] * PAGE + pos % PAGE
        lens = [a + b for a, b in zip(lens, new)]
        qkv = torch.randn(T, (nq + 2 * nkv) * D, device="cuda", generator=_gen(step)).to(torch.bfloat16)
        kvl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        q = ops.rope_and_cache(qkv, pos.to(torch.int32), cs, nq, nkv, slots, k8, v8)
        _check_append(q, k8, v8, qkv, pos.to(torch.int32), cs, slots, nq, nkv, {})
        if new == [1, 1]:
            out = ops.decode_attention(q, k8, v8, kvl, table)
            _check_decode(out, q, k8, v8, table, lens)
        else:
            cu = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
            out = ops.prefill_attention(q, k8, v8, cu, kvl, table, ops.prefill_tiles(new).cuda())
            _check_prefill(out, q, k8, v8, table, new, lens)


def _layer(ops, s):
    q = ops.rope_and_cache(s["qkv"], s["pos"], s["cs"], s["nq"], s["nkv"], s["slots"], s["k8"], s["v8"])
    d = ops.decode_attention(q, s["k8"], s["v8"], s["kvl"], s["table"])
    p = ops.prefill_attention(q, s["k8"], s["v8"], s["cu"], s["kvl"], s["table"], s["tiles"], splits=2)
    return q, d, p


def _layer_state(ops, seed, lens, nq=8, nkv=2):
    k8, v8, kvl, table = _cache(lens, nkv, seed=seed)
    B = len(lens)
    last = kvl.long() - 1
    return dict(nq=nq, nkv=nkv, k8=k8, v8=v8, kvl=kvl, table=table, cs=ops.rope_cos_sin(max(lens), D, 1e4, "cuda"),
                pos=last.to(torch.int32), slots=table.long().gather(1, (last // PAGE)[:, None])[:, 0] * PAGE + last % PAGE,
                qkv=torch.randn(B, (nq + 2 * nkv) * D, device="cuda", generator=_gen(seed)).to(torch.bfloat16),
                cu=torch.arange(B + 1, dtype=torch.int32, device="cuda"), tiles=ops.prefill_tiles([1] * B).cuda())


def test_two_captured_graphs_and_eager_calls_at_once():
    """Two graphs captured on one stream, replayed on two at the same time
    with eager calls on a third: nothing they use is shared."""
    ops = sub("ops")
    states = [_layer_state(ops, 1, [3000, 17, 900]), _layer_state(ops, 2, [5000, 1, 250, 4000]),
              _layer_state(ops, 3, [2500] * 5)]
    want = [_layer(ops, s) for s in states]
    torch.cuda.synchronize()
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for s in states[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(_layer(ops, s))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for round_ in range(20):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graphs[0].replay()
        with torch.cuda.stream(streams[1]):
            graphs[1].replay()
        with torch.cuda.stream(streams[2]):
            eager = _layer(ops, states[2])
        torch.cuda.synchronize()
        for got, w in zip(outs + [eager], want):
            for a, b in zip(got, w):
                assert torch.equal(a, b), f"round {round_}"
    # new inputs in the same buffers
    fresh = _layer_state(ops, 7, [3000, 17, 900])
    for name in ("qkv", "kvl", "table", "pos", "slots"):
        states[0][name].copy_(fresh[name])
    for name in ("k8", "v8"):
        _fill(states[0][name], fresh[name].values, fresh[name].exps)
    graphs[0].replay()
    w = _layer(ops, fresh)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], w))


# ---------------------------------------------------------------- the engine
def _native(cfg, **kw):
    from test_engine_gpu import _engine

    return _engine(cfg, kv_cache_dtype="fp8_e4m3", **kw)


@pytest.mark.parametrize("kw", [dict(), dict(use_graphs=False, mixed_chunk=True), dict(prefill_graph=True),
                                dict(impl="torch")])
def test_native_engine_over_an_8_bit_cache_follows_the_dense_forward(kw):
    """Greedy tokens of prompts across chunks, one of them a prefix-cache hit,
    against the dense fp32 forward whose k and v rows are rounded the same
    way, at the tolerance of the bf16 cache's engine test."""
    from test_engine_gpu import CFG, TOL, _host
    from test_kv8_cpu import _near_argmax

    eng = _native(CFG, prefix_cache=True, **kw)
    w = _host(eng.weights)
    g = torch.Generator().manual_seed(11)
    common = torch.randint(0, CFG.vocab, (48,), generator=g).tolist()
    a, b = (common + torch.randint(0, CFG.vocab, (n,), generator=g).tolist() for n in (30, 9))
    c = torch.randint(0, CFG.vocab, (200,), generator=g).tolist()
    out_a, out_c = eng.generate([a, c], max_new_tokens=6)
    req = eng.add_request(b, 6)
    eng.run()
    assert req.cached_pages == 3
    for p, o in ((a, out_a), (c, out_c), (b, req.output)):
        assert len(o) == 6
        _near_argmax(CFG, w, p, o, TOL)


def test_native_and_oracle_score_text_alike_over_an_8_bit_cache():
    """Per-token logprobs of 400 prompt tokens, native against the fp32 oracle
    on the CPU, both on 8-bit caches; the bf16 cache's bound."""
    from test_engine_gpu import CFG

    models, eng_mod = sub("models"), sub("engine")
    prompt = torch.randint(0, CFG.vocab, (400,), generator=torch.Generator().manual_seed(5)).tolist()
    scores = []
    for kw in (dict(device="cuda"), dict(device="cpu", impl="oracle")):
        w = models.LlamaWeights(CFG, 0, 1, "cpu", seed=0, full_init=True)
        if kw["device"] == "cuda":
            w.embed, w.norm, w.lm_head = w.embed.cuda(), w.norm.cuda(), w.lm_head.cuda()
            w.layers = [{k: v.cuda() for k, v in L.items()} for L in w.layers]
        eng = eng_mod.LLMEngine(CFG, weights=w, max_batch=2, max_seq=512, chunk=128, kv_cache_dtype="fp8_e4m3", **kw)
        r = eng.add_request(prompt, 1, prompt_logprobs=True)
        eng.run()
        scores.append(torch.tensor([x[0] for x in r.prompt_token_logprobs[1:]]))
    assert (scores[0] - scores[1]).abs().mean().item() < 0.05


def _attention_inputs(eng, kv_lens, q_lens, seed):
    cfg = eng.cfg
    k8, v8, kvl, table = _cache(kv_lens, cfg.kv_heads, seed=seed, columns=eng.max_blocks_per_seq)
    q = torch.randn(sum(q_lens), cfg.heads, D, device="cuda", generator=_gen(seed)).to(torch.bfloat16)
    return k8, v8, kvl, table, q


@pytest.mark.parametrize("scratch", [1, 30, 10 ** 6])
def test_engine_prefill_attention_in_groups_of_bounded_scratch(scratch):
    """A batch's attention in as many calls as its scratch bound asks for."""
    from test_engine_gpu import CFG

    ops, launches = sub("ops"), sub("utils.launches")
    eng = _native(CFG, use_graphs=False, max_seq=1024)
    eng.scratch_pages = scratch
    kv_lens, q_lens = [100, 264, 1, 777, 16, 300], [100, 64, 1, 257, 3, 17]
    k8, v8, kvl, table, q = _attention_inputs(eng, kv_lens, q_lens, 4)
    attn = eng._attn_over_fp8(q_lens, kv_lens, table)
    before = launches.get()
    out = attn(0, q, k8, v8)
    calls = {1: 6, 30: 3, 10 ** 6: 1}[scratch]  # pages 7 + 17 + 1, 49, 1 + 19
    assert 2 * calls <= launches.get() - before <= 3 * calls
    _check_prefill(out, q, k8, v8, table, q_lens, kv_lens)
    assert ops.gemm_error() == 0


@pytest.mark.parametrize("scratch", [10, 10 ** 6])
def test_overlapped_halves_of_a_prefill_batch(scratch):
    """The two micro-batches' attention, each on a stream of its own, the
    straddling request cut between them."""
    from test_engine_gpu import CFG

    ops = sub("ops")
    eng = _native(CFG, use_graphs=False, max_seq=1024)
    eng.scratch_pages = scratch
    kv_lens, q_lens = [100, 700, 450], [100, 300, 50]
    k8, v8, kvl, table, q = _attention_inputs(eng, kv_lens, q_lens, 5)
    eng.model.overlap_split = lambda T: 256
    T1, first, second = eng._attn_halves(q_lens, kv_lens, table, 450, eng._attn_over_fp8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        a = first(0, q[:T1], k8, v8)
        with torch.cuda.stream(side), ops.workspace_lane(1):
            b = second(0, q[T1:], k8, v8)
        torch.cuda.synchronize()
        _check_prefill(torch.cat([a, b]), q, k8, v8, table, q_lens, kv_lens)
    assert ops.gemm_error() == 0


def test_prefill_graph_halves_over_an_8_bit_cache():
    """PrefillGraphRunner's two micro-batches, captured on two streams of one
    graph and replayed for chunks of growing context."""
    from test_engine_gpu import CFG

    ops, gr = sub("ops"), sub("engine.graph_runner")
    eng = _native(CFG, use_graphs=False, max_seq=1024)
    T, T1 = 300, 128
    eng.model.overlap_split = lambda n: T1
    runner = gr.PrefillGraphRunner(eng, T)
    seen = {}
    eng.model.forward = lambda *args, attn_halves=None, **kw: seen.update(halves=attn_halves, whole=args[4])
    runner._forward()
    split, first, second = seen["halves"]
    assert split == T1
    k8, v8, _, table, q = _attention_inputs(eng, [500], [T], 6)
    side, lane = torch.cuda.Stream(), torch.cuda.Stream()
    for h in (first, second, seen["whole"]):  # workspaces before the capture
        h(0, q[:T1] if h is first else q[T1:] if h is second else q, k8, v8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        lane.wait_stream(side)
        a = first(0, q[:T1], k8, v8)
        with torch.cuda.stream(lane), ops.workspace_lane(1):
            b = second(0, q[T1:], k8, v8)
        side.wait_stream(lane)
        whole = seen["whole"](0, q, k8, v8)
    runner.bt.copy_(table[:1])
    for n in (300, 417, 500):
        runner.kvl.fill_(n)
        runner.halves[0]["kvl"].fill_(n - (T - T1))
        graph.replay()
        torch.cuda.synchronize()
        _check_prefill(torch.cat([a, b]), q, k8, v8, table, [T], [n])
        _check_prefill(whole, q, k8, v8, table, [T], [n])
    assert ops.gemm_error() == 0


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_second_device_while_the_first_is_current():
    ops = sub("ops")
    s = _layer_state(ops, 1, [300, 17])
    want = _layer(ops, s)
    other = {}
    for k, v in s.items():
        if isinstance(v, torch.Tensor):
            v = v.to("cuda:1")
        elif isinstance(v, ops.Fp8Pages):
            v = ops.Fp8Pages(v.values.to("cuda:1"), v.exps.contiguous().to("cuda:1"))
        other[k] = v
    got = _layer(ops, other)
    torch.cuda.synchronize("cuda:1")
    assert all(torch.equal(a, b.to("cuda:0")) for a, b in zip(want, got))
    with pytest.raises(RuntimeError, match="must be on"):
        ops.decode_attention(want[0], other["k8"], other["v8"], s["kvl"], s["table"])
