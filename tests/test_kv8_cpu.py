"""The 8-bit KV cache's format, its PyTorch statement and its entry points'
refusals (no GPU): a wrong call is refused before anything is launched."""
import glob
import os

import pytest
import torch

from conftest import PKG, ROOT, sub

D, PAGE = 128, 16


def _built():
    return bool(glob.glob(os.path.join(ROOT, PKG, "_C.*.so")))


needs_ext = pytest.mark.skipif(not _built(), reason="_C is not built in this tree")


def _brute(row):
    """Exponent and values of one fp64 row by search over every e4m3 number."""
    b = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    b = b[torch.isfinite(b)].unique()
    top = max(abs(x) for x in row)
    e = -117
    while top > 448 * 2.0 ** e:
        e += 1
    out = []
    for x in row:
        d = (b * 2.0 ** e - x).abs()
        near = b[d == d.min()]
        if near.numel() > 1:  # a tie: the one whose last fraction bit is 0
            near = near[[int(v.to(torch.float8_e4m3fn).view(torch.uint8)) % 2 == 0 for v in near.float()]]
        out.append(float(near[0]) * 2.0 ** e)
    return e, out


def test_rows_are_the_nearest_e4m3_numbers_at_the_smallest_exponent():
    f8 = sub("ops.fp8_pages")
    g = torch.Generator().manual_seed(0)
    x = torch.randn(24, D, generator=g, dtype=torch.float64) * torch.exp2(
        torch.randint(-40, 40, (24, 1), generator=g).double())
    x[0] = 0
    x[1, :4] = torch.tensor([448.0, -432.0, 2.0 ** -9, 2.0 ** -10])          # top exactly 448: exponent 0; ties
    x[1, 4:] = 0
    x[2, 0] = 448.0 * (1 + 2.0 ** -40)                                       # just above: exponent 1
    x[2, 1:] = 1.0
    x[3] = x[3].sign() * 2.0 ** -133                                         # bf16's smallest: held at 2^-117
    x[4, :3] = torch.tensor([400.0, 17 + 2.0 ** -30, 17 - 2.0 ** -30], dtype=x.dtype)  # next to a border, in 64 bits
    x[4, 3:] = 17.0                                                          # the border itself: to even (16)
    values, exps = f8.quantize_rows(x)
    got = f8.dequantize_rows(values, exps).double()
    for i in range(x.shape[0]):
        e, want = _brute(x[i].tolist())
        assert int(exps[i]) == e + 127, i
        assert got[i].tolist() == want, i
    assert int(exps[0]) == 10 and int(exps[1]) == 127 and int(exps[2]) == 128
    assert got[4, 1:4].tolist() == [18.0, 16.0, 16.0]
    # a stored row is exact in bf16
    assert torch.equal(got.to(torch.bfloat16).double(), got)


def test_elements_that_are_not_finite_become_nan_and_leave_the_rest_alone():
    f8 = sub("ops.fp8_pages")
    x = torch.linspace(-3, 3, D).repeat(2, 1)
    y = x.clone()
    y[1, 5], y[1, 9], y[1, 10] = float("inf"), float("nan"), float("-inf")
    a, b = (f8.dequantize_rows(*f8.quantize_rows(t)) for t in (x, y))
    bad = ~torch.isfinite(y)
    assert torch.isnan(b[bad]).all() and torch.equal(b[~bad], a[~bad])


def test_stored_numbers_are_exact_in_bf16_below_2_to_the_128():
    """Every e4m3 number at every exponent byte of the stated range."""
    f8 = sub("ops.fp8_pages")
    v = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    v = v[~torch.isnan(v.float())]
    for byte in range(1, 255):
        real = v.double() * 2.0 ** (byte - 127)
        wide = f8.dequantize_rows(v[None], torch.tensor([byte], dtype=torch.uint8))[0]
        inside = real.abs() < 2.0 ** 128
        assert inside.all() or byte > 246
        assert torch.equal(wide.double()[inside], real[inside])
        assert torch.isinf(wide[~inside]).all()
        half = wide.to(torch.bfloat16).double()
        if byte >= 3:
            assert torch.equal(half[inside], real[inside])
        else:
            assert ((half - real).abs() <= 2.0 ** -134).all()


def test_a_row_at_bf16s_maximum_rounds_up_to_infinity():
    f8 = sub("ops.fp8_pages")
    x = torch.full((1, D), torch.finfo(torch.bfloat16).max)
    values, exps = f8.quantize_rows(x)
    assert int(exps) == 247 and (values.float() == 256).all()
    assert torch.isinf(f8.dequantize_rows(values, exps)).all()


def test_cache_constructor_layout():
    ops = sub("ops")
    k, v = ops.fp8_cache(3, 2, "cpu")
    assert k.shape == (3, 2, PAGE, D) and v.values.dtype == torch.float8_e4m3fn
    assert k.exps.shape == (3, 2, PAGE) and k.exps.stride() == (64, 32, 1)
    assert v.exps.data_ptr() - k.exps.data_ptr() == PAGE
    assert k.dequantize().abs().sum() == 0 and k.device.type == "cpu"


def test_page_plan_packs_pages():
    ops = sub("ops")
    p = ops.page_plan([33, 0, 16, 200], 4)
    assert p.pages == 3 + 0 + 1 + 4
    assert p.table.tolist() == [[0, 1, 2, -1], [-1] * 4, [3, -1, -1, -1], [4, 5, 6, 7]]


def test_oracle_writes_and_reads_the_format():
    """The oracle's cache write and paged attention on an 8-bit cache."""
    ops, oracle, ref, f8 = sub("ops"), sub("ops.oracle"), sub("ops.reference"), sub("ops.fp8_pages")
    torch.manual_seed(0)
    T, nq, nkv = 21, 4, 2
    cs = ops.rope_cos_sin(64, D, 10000.0, "cpu")
    qkv = torch.randn(T, (nq + 2 * nkv) * D).to(torch.bfloat16)
    pos = torch.arange(T, dtype=torch.int32)
    bt = torch.tensor([[2, 0]], dtype=torch.int32)
    slots = bt[0].long()[pos.long() // PAGE] * PAGE + pos.long() % PAGE
    w = (1 + 0.1 * torch.randn(D)).to(torch.bfloat16)
    for norm in ({}, dict(q_norm=w, k_norm=w, eps=1e-5)):
        k8, v8 = ops.fp8_cache(3, nkv, "cpu")
        q = oracle.rope_and_cache(qkv, pos, cs, nq, nkv, slots, k8, v8, **norm)
        k = qkv[:, nq * D:(nq + nkv) * D].view(T, nkv, D).double()
        if norm:
            k = ref.rmsnorm(k, w, 1e-5)
        want, _ = f8.quantize_rows(ref.rope(k, pos, cs))
        got = k8.values.view(torch.uint8)[slots // PAGE, :, slots % PAGE]
        assert torch.equal(got, want.view(torch.uint8))
        kk, vv = ref.gather_kv(k8, bt[0], T), ref.gather_kv(v8, bt[0], T)
        # e4m3 keeps 4 significant bits: half a step is 2^-4 of the value
        v = qkv[:, (nq + nkv) * D:].view(T, nkv, D).float()
        top = v.abs().amax(-1, keepdim=True)
        assert ((vv - v).abs() <= v.abs() * 2.0 ** -4 + top * 2.0 ** -17).all()
        out = oracle.paged_attention(q, k8, v8, [T], [T], bt)
        assert torch.equal(out, ref.attention(q, kk, vv, causal_offset=0).to(q.dtype))


def test_oracle_writes_as_the_kernel_does_outside_the_cache_and_the_table():
    """Slots that are negative or past the cache are not written, the last of
    equal slots stays, positions outside the table take its ends."""
    ops, oracle, f8 = sub("ops"), sub("ops.oracle"), sub("ops.fp8_pages")
    T, nq, nkv, blocks = 40, 2, 2, 3
    g = torch.Generator().manual_seed(0)
    cs = ops.rope_cos_sin(16, D, 10000.0, "cpu")
    qkv = torch.randn(T, (nq + 2 * nkv) * D, generator=g).to(torch.bfloat16)
    pos = torch.randint(-5, 30, (T,), generator=g, dtype=torch.int32)
    slots = torch.randint(0, 12, (T,), generator=g)
    slots[3], slots[4], slots[T - 1] = -1, blocks * PAGE, -17
    k8, v8 = ops.fp8_cache(blocks, nkv, "cpu")
    q = oracle.rope_and_cache(qkv, pos, cs, nq, nkv, slots, k8, v8)
    inside = oracle.rope_and_cache(qkv, pos.clamp(0, 15), cs, nq, nkv)
    assert torch.equal(q, inside)
    last = {s: t for t, s in enumerate(slots.tolist()) if 0 <= s < blocks * PAGE}
    v = qkv[:, (nq + nkv) * D:].view(T, nkv, D).float()
    values, exps = f8.quantize_rows(v)
    rows = v8.values.view(torch.uint8).transpose(1, 2).reshape(-1, nkv, D)
    for s in range(blocks * PAGE):
        if s in last:
            assert torch.equal(rows[s], values[last[s]].view(torch.uint8)), s
            assert torch.equal(v8.exps[s // PAGE, :, s % PAGE], exps[last[s]])
        else:
            assert (rows[s] == 0).all() and (v8.exps[s // PAGE, :, s % PAGE] == 127).all()


def test_page_ids_of_two_threads(monkeypatch):
    """A thread that needs fewer pages appends its list while another makes a
    longer one: each gets as many as it asked for."""
    ops = sub("ops")
    dev = torch.device("cpu")
    monkeypatch.setattr(ops, "_PAGE_IDS", {})

    class Made(list):
        def append(self, t):  # the other thread appends right behind
            super().append(t)
            super().append(torch.arange(5, dtype=torch.int32))

    ops._PAGE_IDS[dev] = Made()
    assert ops._page_ids(9000, dev).tolist() == list(range(9000))
    assert ops._page_ids(20000, dev).tolist() == list(range(20000))
    assert ops._page_ids(3, dev).tolist() == [0, 1, 2]


def _args(ops, T=3, nq=4, nkv=2, blocks=3):
    k, v = ops.fp8_cache(blocks, nkv, "cpu")
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    return dict(
        rope=dict(qkv=bf(T, (nq + 2 * nkv) * D), positions=i32(T), cos_sin=torch.zeros(8, D), nq=nq, nkv=nkv,
                  slots=torch.zeros(T, dtype=torch.int64), k_cache=k, v_cache=v),
        read=dict(k_cache=k, v_cache=v, block_table=i32(T, 2), kv_len=i32(T)),
        decode=dict(q=bf(T, nq, D), k_cache=k, v_cache=v, kv_len=i32(T), block_table=i32(T, 2)))


def _pages(ops, **kw):
    k, _ = ops.fp8_cache(kw.pop("blocks", 3), kw.pop("nkv", 2), "cpu")
    return ops.Fp8Pages(kw.get("values", k.values), kw.get("exps", k.exps))


REFUSED = [
    ("rope", dict(page=32), "16 tokens"),
    ("rope", dict(qkv="float"), "qkv must be"),
    ("rope", dict(nq=3), "qkv must be"),
    ("rope", dict(nkv=0), "qkv must be"),
    ("rope", dict(positions="long"), "positions must be"),
    ("rope", dict(slots="int"), "slots must be"),
    ("rope", dict(cos_sin=torch.zeros(0, D)), "cos_sin must be"),
    ("rope", dict(cos_sin=torch.zeros(8, 64)), "cos_sin must be"),
    ("rope", dict(q_norm=torch.zeros(D, dtype=torch.bfloat16)), "go together"),
    ("rope", dict(q_out=torch.zeros(1, dtype=torch.bfloat16)), "q_out must be"),
    ("read", dict(kv_len="long"), "kv_len must be"),
    ("read", dict(block_table=torch.zeros(2, 2, dtype=torch.int32)), "block_table must be"),
    ("read", dict(k_out=torch.zeros(5, 2, PAGE, D, dtype=torch.bfloat16),
                  v_out=torch.zeros(5, 2, PAGE, D, dtype=torch.bfloat16)), "must hold"),
    ("read", dict(k_out=torch.zeros(6, 2, PAGE, D, dtype=torch.bfloat16),
                  v_out=torch.zeros(6, 2, PAGE, D)), "v_out must be"),
    ("read", dict(k_out=torch.zeros(6, 2, PAGE, D, dtype=torch.bfloat16),
                  v_out=torch.zeros(6, 2, PAGE, D, dtype=torch.bfloat16),
                  out_table=torch.zeros(3, 1, dtype=torch.int32)), "out_table must have"),
    ("decode", dict(q=torch.zeros(3, 4, 64, dtype=torch.bfloat16)), "q must be"),
    ("decode", dict(q=torch.zeros(3, 5, D, dtype=torch.bfloat16)), "q heads"),
    ("decode", dict(q=torch.zeros(3, 34, D, dtype=torch.bfloat16)), "q heads"),
    ("decode", dict(q=torch.zeros(3, 8, D, dtype=torch.bfloat16)[:, ::2]), "contiguous"),
    ("decode", dict(kv_len=torch.zeros(2, dtype=torch.int32)), "kv_len must be"),
    ("decode", dict(block_table=torch.zeros(3, 4, dtype=torch.int32)[:, ::2]), "block_table must be"),
    ("decode", dict(out=torch.zeros(3, 4, D)), "out must be"),
]


def _call(ops, which, a):
    return dict(rope=ops.rope_and_cache, read=ops.read_pages, decode=ops.decode_attention)[which](**a)


@needs_ext
@pytest.mark.parametrize("which,change,message", REFUSED)
def test_refusals(which, change, message):
    ops = sub("ops")
    a = _args(ops)[which]
    for name, v in change.items():
        a[name] = getattr(a[name], v)() if isinstance(v, str) else v
    with pytest.raises((RuntimeError, ValueError), match=message):
        _call(ops, which, a)


@needs_ext
@pytest.mark.parametrize("which", ["rope", "read", "decode"])
def test_refusals_of_the_cache(which):
    ops = sub("ops")
    k, v = ops.fp8_cache(3, 2, "cpu")
    for bad, message in ((ops.Fp8Pages(k.values.view(torch.uint8), k.exps), "float8_e4m3fn"),
                         (ops.Fp8Pages(k.values[:, :, :8], k.exps), "float8_e4m3fn"),
                         (ops.Fp8Pages(k.values[:0], k.exps[:0]), "at least one block"),
                         (ops.Fp8Pages(k.values[:2], k.exps), "exps must be"),
                         (ops.Fp8Pages(k.values, k.exps.float()), "exps must be"),
                         (ops.Fp8Pages(k.values, torch.zeros(3, 2, 24, dtype=torch.uint8)[..., :16]), "exps must be"),
                         (ops.Fp8Pages(k.values.transpose(0, 1), k.exps), "k_cache")):
        a = _args(ops)[which]
        a["k_cache"] = bad
        with pytest.raises(RuntimeError, match=message):
            _call(ops, which, a)
    a = _args(ops)[which]
    a["v_cache"] = _pages(ops, blocks=4)
    with pytest.raises(RuntimeError, match="same shape"):
        _call(ops, which, a)
    a["v_cache"] = torch.zeros(3, 2, PAGE, D, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="both be Fp8Pages"):
        _call(ops, which, a)
    # right in every respect but the device
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        _call(ops, which, _args(ops)[which])


@needs_ext
def test_refused_calls_count_no_launches():
    ops, launches = sub("ops"), sub("utils.launches")
    k, v = ops.fp8_cache(3, 2, "cpu")
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    before = launches.get()
    for which in ("rope", "read", "decode"):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            _call(ops, which, _args(ops)[which])
    for splits in (1, 2):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            ops.prefill_attention(torch.zeros(5, 4, D, dtype=torch.bfloat16), k, v, i32(3), i32(2), i32(2, 3), i32(2, 2),
                                  splits=splits)
    assert launches.get() == before


@needs_ext
def test_refusals_of_head_counts_and_outputs():
    ops = sub("ops")
    a = _args(ops)["rope"]
    a["k_cache"], a["v_cache"] = ops.fp8_cache(3, 1, "cpu")
    with pytest.raises(RuntimeError, match="nkv = 2"):
        ops.rope_and_cache(**a)
    a = _args(ops)["read"]
    with pytest.raises(ValueError, match="go together"):
        ops.read_pages(**a, k_out=torch.zeros(6, 2, PAGE, D, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="give them too"):
        ops.read_pages(**a, out_table=torch.zeros(3, 2, dtype=torch.int32))
    with pytest.raises(TypeError, match="8-bit caches"):
        ops.read_pages(torch.zeros(1), torch.zeros(1), a["block_table"], a["kv_len"])


@needs_ext
def test_refusals_of_prefill_attention():
    ops = sub("ops")
    k, v = ops.fp8_cache(3, 2, "cpu")
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    good = dict(q=bf(5, 4, D), k_cache=k, v_cache=v, cu_q=i32(3), kv_len=i32(2), block_table=i32(2, 3),
                tiles=i32(2, 2))
    plan = ops.PagePlan
    for change, message in ((dict(q=bf(5, 4, 64)), "q must be"), (dict(out=bf(4, 4, D)), "out must have"),
                            (dict(q=bf(5, 3, D)), "multiple of the kv heads"),
                            (dict(k_cache=ops.Fp8Pages(k.values[:2], k.exps)), "exps must be"),
                            (dict(cu_q=i32(2)), "cu_q must be"), (dict(kv_len=i32(2).long()), "kv_len must be"),
                            (dict(block_table=i32(3, 3)), "block_table must be"),
                            (dict(plan=plan(i32(3, 3), 4)), "plan table must be"),
                            (dict(plan=plan(i32(2, 2), 4)), "plan table must be"),
                            (dict(plan=plan(i32(2, 3), -1)), "pages"), (dict(tiles=i32(2, 3)), "tiles must be"),
                            (dict(scale=-1.0), "positive scale"), (dict(scale=float("nan")), "positive scale"),
                            (dict(splits=0), "splits"), ({}, "must be a CUDA tensor")):
        with pytest.raises(RuntimeError, match=message):
            ops.prefill_attention(**{**good, **change})
    with pytest.raises(TypeError, match="both be Fp8Pages"):
        ops.prefill_attention(**{**good, "v_cache": bf(3, 2, PAGE, D)})


@needs_ext
def test_tables_whose_keys_pass_an_int32_are_refused():
    """2^27 columns are 2^31 keys; the largest table below is accepted (up to
    the device check). Untouched pages of the tables take no memory."""
    ops = sub("ops")
    k, v = ops.fp8_cache(3, 1, "cpu")
    i32 = lambda *s: torch.empty(*s, dtype=torch.int32)  # noqa: E731
    bf = lambda *s: torch.empty(*s, dtype=torch.bfloat16)  # noqa: E731
    for cols, message in ((1 << 27, "2\\^27 pages"), ((1 << 27) - 1, "must be a CUDA tensor")):
        bt, q, lens = i32(1, cols), bf(1, 4, D), i32(1)
        with pytest.raises(RuntimeError, match=message):
            ops.decode_attention(q, k, v, lens, bt)
        with pytest.raises(RuntimeError, match=message):
            ops.read_pages(k, v, bt, lens, out_table=bt, k_out=bf(2, 1, PAGE, D), v_out=bf(2, 1, PAGE, D))
        with pytest.raises(RuntimeError, match=message):
            ops.prefill_attention(q, k, v, i32(2), lens, bt, i32(1, 2), plan=ops.PagePlan(bt, 2))


# ---------------------------------------------------------------- the engine on an 8-bit cache
def dense_fp8(cfg, w, tokens):
    """``test_engine_cpu._dense`` (fp32, no cache, no pages) with the rotated k
    and the v rounded to the 8-bit cache's rows: (hidden [T, H], logits)."""
    import torch.nn.functional as F

    ops, ref, f8 = sub("ops"), sub("ops.reference"), sub("ops.fp8_pages")

    def rounded(x):
        return f8.dequantize_rows(*f8.quantize_rows(x))

    T, eps, nq, nkv = len(tokens), cfg.eps, cfg.heads, cfg.kv_heads
    cs = ops.rope_cos_sin(cfg.max_pos, D, cfg.rope_theta, "cpu")
    pos = torch.arange(T)
    res = w.embed.float()[torch.tensor(tokens)]
    for L in w.layers:
        qkv = (ref.rmsnorm(res, L["ln1"], eps) @ L["qkv"].float().t()).view(T, -1, D)
        q, k, v = qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:]
        if cfg.qk_norm:
            q, k = ref.rmsnorm(q, L["q_norm"], eps), ref.rmsnorm(k, L["k_norm"], eps)
        q, k, v = ref.rope(q, pos, cs), rounded(ref.rope(k, pos, cs)), rounded(v)
        res = res + ref.attention(q, k, v, causal_offset=0).reshape(T, nq * D) @ L["o"].float().t()
        g, u = (ref.rmsnorm(res, L["ln2"], eps) @ L["gate_up"].float().t()).chunk(2, dim=-1)
        res = res + (F.silu(g) * u) @ L["down"].float().t()
    h = ref.rmsnorm(res, w.norm, eps)
    return h, h @ w.lm_head.float().t()


def _near_argmax(cfg, w, prompt, out, tol):
    seq = list(prompt)
    for t in out:
        _, logits = dense_fp8(cfg, w, seq)
        assert logits[-1][t] >= logits[-1].max() - tol, (len(seq) - len(prompt), t, int(logits[-1].argmax()))
        seq.append(t)


@pytest.mark.parametrize("qk_norm", [False, True])
def test_engine_prefill_over_an_8_bit_cache_matches_the_dense_forward(qk_norm):
    """The bounds of the bf16 cache's test, against a dense forward whose k
    and v rows are rounded the same way."""
    from test_engine_cpu import CFG, _cos, _engine, _prompt_hidden

    models = sub("models")
    cfg = models.LlamaConfig(**{**CFG.__dict__, "qk_norm": qk_norm})
    prompt = torch.randint(0, cfg.vocab, (150,), generator=torch.Generator().manual_seed(1)).tolist()
    for chunk in (150, 64, 37):
        eng = _engine(cfg, chunk=chunk, kv_cache_dtype="fp8_e4m3")
        assert isinstance(eng.kv.caches[0][0], sub("ops").Fp8Pages)
        got = _prompt_hidden(eng, prompt, chunk)
        want, _ = dense_fp8(cfg, eng.weights, prompt)
        assert _cos(got, want[-1]) > 0.999, chunk
        assert float((got - want[-1]).abs().max()) < 0.05 * float(want[-1].abs().max()), chunk


def test_engine_generates_over_an_8_bit_cache():
    """Chunks, batches, a prefix-cache hit and mixed chunks."""
    from test_engine_cpu import CFG, LOGIT_TOL, _engine

    g = torch.Generator().manual_seed(2)
    common = torch.randint(0, CFG.vocab, (48,), generator=g).tolist()
    prompts = [common + torch.randint(0, CFG.vocab, (n,), generator=g).tolist() for n in (30, 1)] + \
        [torch.randint(0, CFG.vocab, (70,), generator=g).tolist()]
    eng = _engine(chunk=32, kv_cache_dtype="fp8_e4m3", prefix_cache=True, mixed_chunk=True)
    first = eng.generate(prompts[:1], max_new_tokens=5)
    outs = first + eng.generate(prompts[1:], max_new_tokens=5)
    assert eng.prefix_cache.hits == 3
    for p, o in zip(prompts, outs):
        assert len(o) == 5
        _near_argmax(CFG, eng.weights, p, o, LOGIT_TOL)


def test_cache_dtype_names_and_sizes():
    from test_engine_cpu import _engine

    kv = sub("engine.kv_cache")
    assert kv.kv_dtype("auto") == kv.kv_dtype("bfloat16") == torch.bfloat16
    assert kv.kv_dtype("fp8_e4m3") == kv.kv_dtype(torch.float8_e4m3fn) == torch.float8_e4m3fn
    for bad in ("fp8_e5m2", "int8", torch.float16, None, 8):
        with pytest.raises(ValueError, match="KV cache dtype"):
            kv.kv_dtype(bad)
    with pytest.raises(ValueError, match="KV cache dtype"):
        _engine(kv_cache_dtype="fp16")
    # 8B: 129 bytes per row instead of 256
    assert kv.PagedKVCache.bytes_per_token(32, 8, 128, 1) == 32 * 2 * 8 * 129
    c = kv.PagedKVCache(2, 2, 128, 5, "cpu", torch.float8_e4m3fn)
    per_block = sum(t.numel() for k, v in c.caches for t in (k.values, v.values, k.exps, v.exps)) // 5
    assert per_block == kv.PagedKVCache.bytes_per_token(2, 2, 128, 1) * kv.PAGE
    with pytest.raises(ValueError, match="head_dim 128"):
        kv.PagedKVCache(1, 2, 64, 5, "cpu", torch.float8_e4m3fn)
    p = sub("server.cli").build_parser()
    assert p.parse_args(["--kv-cache-dtype", "fp8_e4m3"]).kv_cache_dtype == "fp8_e4m3"


def _bare_engine(**kw):
    """An engine's sizes without weights or a cache."""
    eng_mod, models = sub("engine"), sub("models")
    e = object.__new__(eng_mod.LLMEngine)
    e.cfg = models.LlamaConfig(**{**models.LlamaConfig.tiny().__dict__, "heads": 32, "kv_heads": 8})
    e.kv_cache_dtype, e.tp_size, e.overlap = torch.float8_e4m3fn, 1, False
    e.max_batch, e.max_blocks_per_seq, e.scratch_pages = 64, 512, 16384
    e.__dict__.update(kw)
    return e


def test_prefill_scratch_is_bounded_and_counted_in_the_memory_fraction():
    """However many requests share a prefix, a call reads back no more than its
    bound, and the cache leaves that much of the memory fraction free."""
    kv = sub("engine.kv_cache")
    e = _bare_engine(scratch_pages=20)
    assert e._prefill_groups([1]) == [(0, 1)]
    assert e._prefill_groups([160, 160, 16]) == [(0, 2), (2, 3)]
    assert e._prefill_groups([16] * 20) == [(0, 20)] and e._prefill_groups([17] * 20) == [(0, 10), (10, 20)]
    assert e._prefill_groups([9999, 5, 9999]) == [(0, 1), (1, 2), (2, 3)]
    for lens in ([3, 400, 20, 20, 300, 1, 17], [320] * 5):
        groups = e._prefill_groups(lens)
        assert [i for a, b in groups for i in range(a, b)] == list(range(len(lens)))
        assert all(b - a == 1 or sum(-(-n // PAGE) for n in lens[a:b]) <= 20 for a, b in groups)
    # 8 kv heads: 64 KB a page of one layer's keys and values in bf16
    page = kv.PagedKVCache.scratch_bytes(1, 8, 128)
    assert page == 2 * 8 * 16 * 128 * 2
    assert _bare_engine(kv_cache_dtype=torch.bfloat16)._scratch_reserve(True) == 0
    assert _bare_engine()._scratch_reserve(False) == 16384 * page                  # the bound: 64 x 512 pages are more
    assert _bare_engine(max_batch=2)._scratch_reserve(False) == 2 * 512 * page     # all that a batch can need
    assert _bare_engine()._scratch_reserve(True) == (16384 + 512) * page
    assert _bare_engine(overlap=True)._scratch_reserve(True) == 2 * (16384 + 512) * page
    assert _bare_engine(overlap=True, max_batch=2)._scratch_reserve(False) == 3 * 512 * page
    GB = 1 << 30
    assert kv.PagedKVCache.blocks_for_memory(180 * GB, 164 * GB, 0.9, 1 << 20, GB) == \
        kv.PagedKVCache.blocks_for_memory(180 * GB, 164 * GB, 0.9, 1 << 20) - 1024


def test_overlapped_halves_over_an_8_bit_cache_cut_as_over_bf16():
    """The micro-batches' requests, lengths and table rows, as given to the
    8-bit cache's attention."""
    import types

    e = _bare_engine(model=types.SimpleNamespace(overlap_split=lambda T: 256, scale=0.1), device=torch.device("cpu"))
    bt = torch.arange(3 * 8, dtype=torch.int32).view(3, 8)
    got = []
    T1, a, b = e._attn_halves([100, 300, 50], [100, 700, 1050], bt, 450, lambda *args: got.append(args) or len(got))
    assert (T1, a, b) == (256, 1, 2)
    assert got[0][:2] == ([100, 156], [100, 700 - 144]) and torch.equal(got[0][2], bt[[0, 1]])
    assert got[1][:2] == ([144, 50], [700, 1050]) and torch.equal(got[1][2], bt[[1, 2]])


def _tp_worker(rank, world):
    from test_engine_cpu import CFG

    eng_mod, par = sub("engine"), sub("parallel")
    tp = par.TPGroup(None, "cpu", use_mailbox=False)
    eng = eng_mod.LLMEngine(CFG, tp=tp, impl="oracle", device="cpu", full_init=True, seed=0, max_batch=4, max_seq=512,
                            chunk=32, kv_cache_dtype="fp8_e4m3", mixed_chunk=True)
    assert eng.kv.caches[0][0].shape[1] == CFG.kv_heads // world
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, CFG.vocab, (n,), generator=g).tolist() for n in (70, 9, 33)]
    return {"prompts": prompts, "out": eng.generate(prompts, max_new_tokens=4)}


def test_two_tensor_parallel_ranks_over_an_8_bit_cache():
    from _mp import run_ranks
    from test_engine_cpu import CFG, LOGIT_TOL

    models = sub("models")
    res = run_ranks(_tp_worker, 2)
    assert res[0] == res[1]
    w = models.LlamaWeights(CFG, 0, 1, "cpu", seed=0, full_init=True)  # the same model, unsharded
    for p, o in zip(res[0]["prompts"], res[0]["out"]):
        assert len(o) == 4
        _near_argmax(CFG, w, p, o, LOGIT_TOL)
