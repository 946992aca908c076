"""Serving from a key-value cache kept in 8 bits: the cases of its operators.

A cached row (128 head dimensions of one token and one key-value head) is held
as e4m3 numbers with one power-of-two scale: ``row = values * 2^(exps - 127)``,
the exponent the smallest one at which the row's largest magnitude is at most
448 (never below 2^-117). A power of two only moves exponents, so a stored row
times its scale is exact in bfloat16. Pages hold 16 tokens:
``values [blocks, kv heads, 16, 128]`` e4m3, ``exps [blocks, kv heads, 16]``
uint8, one pair for the keys and one for the values.

Four operators, each with the sizes it is used at:

* append:  rotary embedding of q and k of a fused projection, k and v rounded
           into the cache; the pages that were written are read back
* read:    pages of a ragged batch back to bfloat16
* decode:  attention of one new token per request over the cache
* prefill: causal attention of a prompt's chunk over the cache

Rows behind a request's length hold garbage (NaN bytes) here, as reused pages
do in a server. ``run`` gives the plain form, or with ``own`` the calls of
``mailbox_ar_b200.ops``.
"""
import math

import torch

own = False

PAGE, D = 16, 128
THETA, EPS = 500000.0, 1e-5


def listed():
    return [
        # one request's next token, 8B heads: latency only
        dict(name="append_token", op="append", R=1, nq=32, nkv=8, start=4095, new=1, norm=False),
        # a decode batch whose q and k are normalised per head
        dict(name="append_batch_norm", op="append", R=64, nq=32, nkv=8, start=1037, new=1, norm=True),
        # a prefill chunk that starts inside a page
        dict(name="append_chunk", op="append", R=1, nq=32, nkv=8, start=1029, new=1024, norm=False),
        # several prompts in one 70B batch
        dict(name="append_prompts", op="append", R=5, nq=64, nkv=8, start=0, new=1601, norm=False),
        # a shared prefix of odd length
        dict(name="read_prefix", op="read", R=1, nkv=8, ctx=777, ragged=False),
        # a ragged batch of long requests
        dict(name="read_batch", op="read", R=37, nkv=8, ctx=8192, ragged=True),
        # the first token after a one-token prompt: the smallest call
        dict(name="decode_first", op="decode", R=1, nq=32, nkv=8, ctx=1, ragged=False),
        # one request at the decode benchmark's context
        dict(name="decode_one", op="decode", R=1, nq=32, nkv=8, ctx=4096, ragged=False),
        # a full ragged batch up to the default longest request
        dict(name="decode_batch", op="decode", R=64, nq=32, nkv=8, ctx=8192, ragged=True),
        # one rank of eight of a 70B model, few requests of long context
        dict(name="decode_long_rank", op="decode", R=8, nq=8, nkv=1, ctx=131072, ragged=False),
        # a chunk of a long prompt
        dict(name="prefill_chunk", op="prefill", R=1, nq=32, nkv=8, ctx=8192, new=1024, ragged=False),
        # a ragged batch of short pieces on one rank of eight
        dict(name="prefill_ragged_rank", op="prefill", R=7, nq=8, nkv=1, ctx=2049, new=333, ragged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "read", "decode", "prefill"))
    nkv = rng.choice((1, 2, 4, 8))
    nq = nkv * rng.choice((1, 3, 4, 7, 8, 16))
    if op == "append":
        R = _log(rng, 1, 64)
        new = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, 4000 // R))
        return dict(op=op, R=R, nq=nq, nkv=nkv, start=rng.randrange(0, 5000), new=new, norm=rng.random() < 0.4)
    ctx = _log(rng, 1, 65536 if op == "decode" else 9000)
    R = _log(rng, 1, max(1, min(96, (150000 if op == "read" else 260000) // ctx)))
    if op == "read":
        return dict(op=op, R=R, nkv=nkv, ctx=ctx, ragged=rng.random() < 0.6)
    if op == "decode":
        return dict(op=op, R=R, nq=nq, nkv=nkv, ctx=ctx, ragged=rng.random() < 0.6)
    nq, ctx = min(nq, nkv * 8, 32), min(ctx, 8000)
    nq -= nq % nkv
    new = _log(rng, 1, min(ctx, 1024))
    R = max(1, min(R, 6_000_000 // (new * ctx)))
    return dict(op=op, R=R, nq=nq, nkv=nkv, ctx=ctx, new=new, ragged=rng.random() < 0.6)


def _lens(case):
    """Lengths of the requests: the whole context, or spread over it with one
    request at it (and, of eight or more that need not hold a token, one empty)."""
    if case["op"] == "append":
        return [case["start"] + case["new"]] * case["R"]
    R, ctx = case["R"], case["ctx"]
    if not case["ragged"]:
        return [ctx] * R
    lens = [1 + ((r * 7919 + 104729) * 2654435761 % (1 << 32)) * ctx // (1 << 32) for r in range(R)]
    lens[0] = ctx
    if R >= 8 and case["op"] != "prefill":
        lens[3] = 0
    return lens


def _q_lens(case):
    return [min(n, case["new"]) for n in _lens(case)]


def _pages(n):
    return -(-n // PAGE)


def work(case):
    lens, nkv, nq = _lens(case), case["nkv"], case.get("nq", 0)
    row = nkv * 2 * (D + 1)  # a token's k and v rows and their exponents
    if case["op"] == "append":
        T = case["R"] * case["new"]
        first = case["start"] % PAGE
        back = case["R"] * (first + case["new"])  # rows of the touched pages
        return {"bytes": T * ((nq + 2 * nkv) * D * 2 + nq * D * 2 + D * 4 + row + 12) + back * (row + nkv * 2 * D * 2),
                "flops": T * (nq + nkv) * D * 3}
    if case["op"] == "read":
        return {"bytes": sum(lens) * (row + nkv * 2 * D * 2), "flops": sum(lens) * nkv * 2 * D}
    if case["op"] == "decode":
        return {"bytes": sum(lens) * row + 2 * case["R"] * nq * D * 2 + 4 * sum(map(_pages, lens)),
                "flops": 4 * nq * D * sum(lens)}
    q = _q_lens(case)
    pairs = sum(n * (2 * L - n + 1) // 2 for n, L in zip(q, lens))
    return {"bytes": sum(lens) * row + 2 * sum(q) * nq * D * 2, "flops": 4 * nq * D * pairs}


# ---------------------------------------------------------------- inputs
def _quantise(x):
    """e4m3 rows and their exponents (biased by 127) of x [..., 128], at x's precision."""
    m, e = torch.frexp(x.abs().amax(-1))
    e = torch.where(m > 0.875, e - 8, e - 9)  # 448 = 0.875 * 2^9
    e = torch.where(m == 0, torch.full_like(e, -117), e.clamp_min(-117))
    y = torch.ldexp(x, -e.unsqueeze(-1))
    # to 4 significant bits at x's precision first (2^-9 is the smallest step): one rounding, ties to even
    step = torch.frexp(y)[1].clamp_min(-5) - 4
    y = torch.ldexp(torch.round(torch.ldexp(y, -step)), step)
    return y.to(torch.float32).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _rope_table(n, device):
    inv = 1.0 / THETA ** (torch.arange(0, D, 2, dtype=torch.float64, device=device) / D)
    ang = torch.arange(n, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([ang.cos(), ang.sin()], 1).float()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g)

    lens, nkv = _lens(case), case["nkv"]
    R, per = case["R"], _pages(max(max(lens), 1))
    counts = [_pages(n) for n in lens]
    blocks = sum(counts) + 2
    # pages of the requests scattered over the cache; entries behind a request's pages name page 0
    perm = torch.randperm(blocks, device=dev, generator=g).to(torch.int32)
    kv_len = torch.tensor(lens, dtype=torch.int32, device=dev)
    ends = torch.tensor(counts, device=dev).cumsum(0)
    i = torch.arange(per, device=dev)[None, :]
    used = i < torch.tensor(counts, device=dev)[:, None]
    flat = (ends[:, None] - torch.tensor(counts, device=dev)[:, None] + i).clamp_max(blocks - 1)
    table = torch.where(used, perm[flat], torch.zeros((), dtype=torch.int32, device=dev)).contiguous()
    # keys with a few strong channels, as trained models have them; garbage where no token lives
    old = torch.tensor(lens, device=dev) if case["op"] != "append" else torch.full((R,), case["start"], device=dev)
    live = torch.zeros(blocks, PAGE, dtype=torch.bool, device=dev)
    rows = (old[:, None] - i * PAGE).clamp(0, PAGE)
    live[table[used].long()] = torch.arange(PAGE, device=dev)[None, :] < rows[used][:, None]
    cache = []
    for strong in (4.0, 1.0):
        x = randn(blocks, nkv, PAGE, D)
        x[..., ::17] *= strong
        v8, e8 = _quantise(x)
        v8 = torch.where(live[:, None, :, None], v8.view(torch.uint8), 0x7F).view(torch.float8_e4m3fn)
        e8 = torch.where(live[:, None, :], e8, 0xFF)
        cache += [v8, e8]
    s = dict(case=dict(case), kv_len=kv_len, table=table, cache=cache)
    if case["op"] == "append":
        new, start, nq = case["new"], case["start"], case["nq"]
        pos = start + torch.arange(new, device=dev)
        s["positions"] = pos.to(torch.int32).repeat(R)
        s["slots"] = (table.long()[:, pos // PAGE] * PAGE + pos % PAGE).reshape(-1)
        s["qkv"] = randn(R * new, (nq + 2 * nkv) * D).to(torch.bfloat16)
        s["cos_sin"] = _rope_table(start + new, dev)
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = ((1 + 0.2 * randn(D)).to(torch.bfloat16) for _ in range(2))
        # the pages that get written, as tables and lengths of their own
        s["table"] = table[:, start // PAGE:].contiguous()
        s["kv_len"] = torch.full((R,), start % PAGE + new, dtype=torch.int32, device=dev)
    if case["op"] in ("append", "read"):
        n = s["table"].numel()
        s["out"] = [torch.zeros(n, nkv, PAGE, D, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    if case["op"] == "decode":
        s["q"] = randn(R, case["nq"], D).to(torch.bfloat16)
    if case["op"] == "prefill":
        q_lens = _q_lens(case)
        s["q"] = randn(sum(q_lens), case["nq"], D).to(torch.bfloat16)
        s["cu_q"] = torch.tensor([0] + q_lens, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)
        tiles = sorted(((r, o) for r, n in enumerate(q_lens) for o in range(0, n, 256)), key=lambda t: -t[1])
        s["tiles"] = torch.tensor(tiles, dtype=torch.int32).reshape(-1, 2).to(dev)
        s["new"] = max(q_lens)
    return s


# ---------------------------------------------------------------- plain form
def _dequant(v8, e8):
    return torch.ldexp(v8.float(), e8[..., None].int() - 127)


def _rope(x, pos, cos_sin):
    cs = cos_sin[pos.long()][:, None].to(x.dtype)
    c, s = cs[..., :D // 2], cs[..., D // 2:]
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _norm(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.to(x.dtype)


def _read(s):
    """Pages of every request, requests one after another; rows behind a
    length are zeros, pages behind it stay as they were."""
    kv, n = s["kv_len"], s["table"].shape[1]
    i = torch.arange(n * PAGE, device=kv.device).view(1, n, PAGE)
    live = i < kv[:, None, None]
    at = live.any(-1).reshape(-1)
    for out, (v8, e8) in zip(s["out"], (s["cache"][:2], s["cache"][2:])):
        x = _dequant(v8.view(torch.uint8)[s["table"].long()].view(torch.float8_e4m3fn), e8[s["table"].long()])
        x = torch.where(live[:, :, None, :, None], x, torch.zeros((), device=x.device)).flatten(0, 1)
        out.copy_(torch.where(at[:, None, None, None], x.to(out.dtype), out))
    return s["out"]


def _gather(s, which):
    """[R, kv heads, pages * 16, 128] of the requests, zeros behind their lengths."""
    v8, e8 = s["cache"][2 * which:2 * which + 2]
    t = s["table"].long()
    x = _dequant(v8.view(torch.uint8)[t].view(torch.float8_e4m3fn), e8[t]).transpose(1, 2).flatten(2, 3)
    live = torch.arange(x.shape[2], device=x.device)[None, :] < s["kv_len"][:, None]
    return torch.where(live[:, None, :, None], x, torch.zeros((), device=x.device))


def _attend(q, k, v, last):
    """q [R, kv heads, rows, 128] over k, v [R, kv heads, L, 128]; row i sees
    keys 0..last[i]; a row that sees none gives zeros."""
    s = q @ k.transpose(-1, -2) / math.sqrt(D)
    s.masked_fill_(torch.arange(k.shape[2], device=q.device) > last[..., None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp_min(torch.finfo(s.dtype).min)
    p = torch.exp(s.sub_(m))
    return (p @ v) / p.sum(-1, keepdim=True).clamp_min(torch.finfo(s.dtype).tiny)


def run(s):
    c, (kv, ke, vv, ve) = s["case"], s["cache"]
    op, nkv = c["op"], c["nkv"]
    if own:
        from mailbox_ar_b200 import ops

        k8, v8 = ops.Fp8Pages(kv, ke), ops.Fp8Pages(vv, ve)
        if op == "append":
            q = ops.rope_and_cache(s["qkv"], s["positions"], s["cos_sin"], c["nq"], nkv, s["slots"], k8, v8,
                                   q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS)
            k, v = ops.read_pages(k8, v8, s["table"], s["kv_len"], k_out=s["out"][0], v_out=s["out"][1])
            return q, k, v
        if op == "read":
            return ops.read_pages(k8, v8, s["table"], s["kv_len"], k_out=s["out"][0], v_out=s["out"][1])
        if op == "decode":
            return ops.decode_attention(s["q"], k8, v8, s["kv_len"], s["table"])
        splits = ops.prefill_splits(s["tiles"].shape[0], c["nq"], c["ctx"])
        return ops.prefill_attention(s["q"], k8, v8, s["cu_q"], s["kv_len"], s["table"], s["tiles"], splits=splits)
    if op == "append":
        T, nq = s["qkv"].shape[0], c["nq"]
        x = s["qkv"].view(T, nq + 2 * nkv, D)
        q, k, v = x[:, :nq].float(), x[:, nq:nq + nkv].double(), x[:, nq + nkv:].float()  # k: it is rounded to few bits
        if c["norm"]:
            q, k = _norm(q, s["q_norm"]), _norm(k, s["k_norm"])
        q = _rope(q, s["positions"], s["cos_sin"]).to(torch.bfloat16)
        blk, off = s["slots"] // PAGE, s["slots"] % PAGE
        for x, v8, e8 in ((_rope(k, s["positions"], s["cos_sin"]), kv, ke), (v, vv, ve)):
            a, b = _quantise(x)
            v8.view(torch.uint8)[blk, :, off] = a.view(torch.uint8)
            e8[blk, :, off] = b
        return (q, *_read(s))
    if op == "read":
        return tuple(_read(s))
    k, v, q = _gather(s, 0), _gather(s, 1), s["q"]
    R, G = k.shape[0], c["nq"] // nkv
    if op == "decode":
        last = (s["kv_len"] - 1)[:, None, None].expand(R, nkv, G)
        return _attend(q.float().view(R, nkv, G, D), k, v, last).reshape(R, c["nq"], D).to(q.dtype)
    # prefill: the requests' rows padded to the longest, and back
    n, i = s["cu_q"].diff()[:, None], torch.arange(s["new"], device=q.device)[None, :]
    inside = i < n
    x = q[(s["cu_q"][:-1, None] + i.minimum(n - 1)).long()].float()  # [R, new, nq, 128]
    x = x.view(R, s["new"], nkv, G, D).permute(0, 2, 3, 1, 4).flatten(2, 3)
    last = (s["kv_len"][:, None] - n + i)[:, None, None, :].expand(R, nkv, G, s["new"]).flatten(2, 3)
    o = _attend(x, k, v, last).view(R, nkv, G, s["new"], D).permute(0, 3, 1, 2, 4).reshape(R, s["new"], c["nq"], D)
    return o[inside].to(q.dtype)


# ---------------------------------------------------------------- the definition in 64 bits
def _e4m3_rows(x):
    """The e4m3 rows nearest to x (ties to even) at their power-of-two scale, as values."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp_min(1e-300))).long() - 9
    for _ in range(3):
        e = torch.where(top > 448 * torch.exp2(e.double()), e + 1, e)
    y = x * torch.exp2(-e.clamp_min(-117).double())
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step * torch.exp2(e.clamp_min(-117).double())


def _e4m3_values(b):
    """What e4m3 bytes stand for, from their sign, exponent and fraction."""
    b = b.view(torch.uint8).long()
    e, f = (b >> 3) & 15, (b & 7).double()
    x = torch.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * torch.exp2(e.double() - 7))
    return torch.where(b >= 128, -x, x)


def _request(s, which, r, n):
    """[n, kv heads, 128] of request r in 64 bits."""
    t = s["table"][r, :_pages(n)].long()
    x = _e4m3_values(s["cache"][2 * which][t]) * torch.exp2(s["cache"][2 * which + 1][t].double() - 127)[..., None]
    return x.transpose(1, 2).reshape(-1, x.shape[1], D)[:n]


def exact(case, seed):
    s = prepare(case, seed)
    op, nkv, R = case["op"], case["nkv"], case["R"]
    if op == "append":
        nq, T = case["nq"], s["qkv"].shape[0]
        x = s["qkv"].double().view(T, -1, D)
        if case["norm"]:
            w = torch.cat([s["q_norm"].double().expand(nq, D), s["k_norm"].double().expand(nkv, D),
                           torch.ones(nkv, D, dtype=torch.float64, device=x.device)])
            y = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / D + EPS) * w
            x = torch.cat([y[:, :nq + nkv], x[:, nq + nkv:]], 1)
        z = torch.complex(x[:, :nq + nkv, :D // 2], x[:, :nq + nkv, D // 2:])
        cs = s["cos_sin"].double()[s["positions"].long()]
        z = z * torch.complex(cs[:, :D // 2], cs[:, D // 2:])[:, None]
        rot = torch.cat([z.real, z.imag], -1)
        outs, first, new = [], case["start"] % PAGE, case["new"]
        for which, rows in ((0, rot[:, nq:]), (1, x[:, nq + nkv:])):
            rows = _e4m3_rows(rows).view(R, new, nkv, D)
            out = torch.zeros(R, s["table"].shape[1] * PAGE, nkv, D, dtype=torch.float64, device=x.device)
            for r in range(R):
                out[r, :first] = _request(s, which, r, first)
            out[:, first:first + new] = rows
            outs.append(out.view(-1, PAGE, nkv, D).transpose(1, 2).contiguous())
        return (rot[:, :nq], *outs)
    lens = _lens(case)
    if op == "read":
        outs = []
        for which in (0, 1):
            out = torch.zeros(R, s["table"].shape[1] * PAGE, nkv, D, dtype=torch.float64, device="cuda")
            for r, n in enumerate(lens):
                out[r, :n] = _request(s, which, r, n)
            outs.append(out.view(-1, PAGE, nkv, D).transpose(1, 2).contiguous())
        return tuple(outs)
    q = s["q"].double()
    G, out, row = case["nq"] // nkv, torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), 0
    for n, new, r in zip(lens, [1] * R if op == "decode" else _q_lens(case), range(R)):
        if n:
            k, v = _request(s, 0, r, n), _request(s, 1, r, n)
            hidden = torch.arange(n, device="cuda")[None, :] > torch.arange(n - new, n, device="cuda")[:, None]
            for h in range(case["nq"]):
                t = (q[row:row + new, h] @ k[:, h // G].T * D ** -0.5).masked_fill_(hidden, -math.inf)
                out[row:row + new, h] = torch.softmax(t, -1) @ v[:, h // G]
        row += new
    return out
