"""The operators that carry a model of this package one token at a time, as calls to be timed and compared.

  attend     attention of one new token a row over a paged key / value cache (basal::paged_attention)
  append     new tokens' keys and values into the cache's pages (basal::kv_append)
  copy       pages copied within the cache, every layer at once: a fork's or a compaction's moves (basal::kv_copy_pages)
  gdn        the Gated DeltaNet's step for one token a row, its state and convolution inputs updated in place
             (basal::gdn_step)
  constrain  penalties for repeated tokens, biases and grammar masks on a step's logits (basal::constrain_logits)

`own` False computes them in their plain form (elementary torch operations in 32 bits), True calls the package. Layouts:
  pages      k, v [pages, kv heads, page size, d] bf16, fp16 or e4m3; e4m3 pages have a 32-bit scale for each token and
             head, [pages, kv heads, page size]: a value is code * scale, scale = max(amax, 1e-12) / 448
  table      [rows, width] int32: the page that holds positions j * page size ..  of a row; entries that no position
             of the row needs are -1
  lengths    [rows] int32, the new token's own position included; 0 is a row of padding
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # one conversation, a short context: the call's latency is all there is
        dict(name="attend 1 x 200", kind="attend", rows=1, heads=16, kv_heads=4, d=128, page=64, most=200, window=0,
             empty=False, dtype="bf16", fp8=False),
        # a serving batch of uneven rows, one of them padding, the hybrid classifier's heads
        dict(name="attend 64 x 8192", kind="attend", rows=64, heads=16, kv_heads=4, d=128, page=64, most=8192, window=0,
             empty=True, dtype="bf16", fp8=False),
        # two long documents: few rows, the cache's length is what can be spread
        dict(name="attend 2 x 131072", kind="attend", rows=2, heads=16, kv_heads=4, d=128, page=128, most=131072,
             window=0, empty=False, dtype="bf16", fp8=False),
        # 8-bit pages, many rows, eight kv heads
        dict(name="attend fp8 128 x 4001", kind="attend", rows=128, heads=32, kv_heads=8, d=128, page=32, most=4001,
             window=0, empty=True, dtype="bf16", fp8=True),
        # a step's new token for every row of a batch
        dict(name="append 64 x 1", kind="append", rows=64, tokens=1, kv_heads=4, d=128, page=64, before=4000,
             dtype="bf16", fp8=False),
        # prompts of uneven lengths into 8-bit pages
        dict(name="append fp8 16 x 2048", kind="append", rows=16, tokens=2048, kv_heads=4, d=128, page=64, before=100,
             dtype="bf16", fp8=True),
        # the last, half-filled page of one row that is forked: every attention layer of the hybrid classifier
        dict(name="copy 1 page", kind="copy", layers=8, pages=64, moves=1, kv_heads=4, d=128, page=64, fp8=False),
        # the pages of a batch moved together after rows have ended
        dict(name="copy 400 pages", kind="copy", layers=8, pages=900, moves=400, kv_heads=4, d=128, page=64, fp8=False),
        # the hybrid classifier's recurrent layer, one conversation and a serving batch whose rows sit anywhere in the
        # pool of states
        dict(name="gdn 1 row", kind="gdn", rows=1, slots=1, key_heads=16, value_heads=32, dtype="bf16"),
        dict(name="gdn 256 rows", kind="gdn", rows=256, slots=300, key_heads=16, value_heads=32, dtype="bf16"),
        # an answer's next token under a grammar that leaves few tokens, and a batch with open ones
        dict(name="constrain 1 x 151936", kind="constrain", rows=1, vocab=151936, history=300, biases=16, open=0.001,
             dtype="bf16"),
        dict(name="constrain 256 x 151936", kind="constrain", rows=256, vocab=151936, history=2000, biases=64, open=0.5,
             dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "copy", "gdn", "gdn", "constrain"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "attend":
        d = rng.choice([64, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4, 5, 7, 8, 16])
        rows = _log(rng, 1, 160)
        most = _log(rng, 1, min(131072, (1 << 28) // (rows * kv * d)))
        window = rng.choice([0, 0, 0, _log(rng, 1, 4096)])
        return dict(kind=kind, rows=rows, heads=heads, kv_heads=kv, d=d, page=rng.choice([16, 32, 64, 128, 24, 1, 256]),
                    most=most, window=window, empty=rows > 1 and rng.random() < 0.5, dtype=dtype,
                    fp8=rng.random() < 0.4)
    if kind == "append":
        kv = rng.choice([1, 2, 4, 8])
        rows, d = _log(rng, 1, 128), rng.choice([64, 128, 256])
        tokens = rng.choice([1, _log(rng, 1, 2048)])
        tokens = max(1, min(tokens, (1 << 25) // (rows * kv * d)))
        return dict(kind=kind, rows=rows, tokens=tokens, kv_heads=kv, d=d, page=rng.choice([16, 32, 64, 128, 24]),
                    before=_log(rng, 1, 3000), dtype=dtype, fp8=rng.random() < 0.5)
    if kind == "copy":
        pages = _log(rng, 8, 800)
        return dict(kind=kind, layers=rng.choice([1, 2, 6, 8]), pages=pages, moves=rng.randint(1, pages // 2),
                    kv_heads=rng.choice([1, 2, 4]), d=rng.choice([64, 128]), page=rng.choice([16, 64, 24]),
                    fp8=rng.random() < 0.5)
    if kind == "gdn":
        hk = rng.choice([1, 2, 4, 8, 16])
        hv = hk * rng.choice([1, 2, 3, 4] if hk < 16 else [1, 2])
        rows = _log(rng, 1, 200)
        return dict(kind=kind, rows=rows, slots=rows + rng.randint(0, 20), key_heads=hk, value_heads=hv, dtype=dtype)
    return dict(kind=kind, rows=_log(rng, 1, 160), vocab=rng.choice([151936, 32003, _log(rng, 300, 200000)]),
                history=_log(rng, 1, 4000), biases=_log(rng, 1, 200), open=rng.choice([0.0002, 0.01, 0.3, 1.0]),
                dtype=rng.choice(["bf16", "fp16", "fp32"]))


def _lengths(case):
    """Rows' lengths, spread over 1 .. most: the last is the longest, the first is a row of padding where asked."""
    n, most = case["rows"], case["most"]
    got = [1 + int((i * 0.6180339887498949) % 1.0 * most) for i in range(1, n)] + [most]
    if case["empty"]:
        got[0] = 0
    return got


def _counts(case):
    """Tokens that each row of an append brings, and where they begin."""
    n, T = case["rows"], case["tokens"]
    count = [max(1, T - int((i * 0.6180339887498949) % 1.0 * T * 0.6)) for i in range(n)]
    start = [int((i * 0.7548776662466927) % 1.0 * case["before"]) for i in range(n)]
    return count, start


def _tables(ends, begins, page, gen):
    """A table [rows, width] whose pages lie anywhere in a pool, -1 where a row holds nothing, and the pool's pages."""
    need = [[j for j in range((e + page - 1) // page) if (j + 1) * page > b] for e, b in zip(ends, begins)]
    total = sum(map(len, need)) + 3
    width = max(1, max((e + page - 1) // page for e in ends))
    spread = torch.randperm(total, generator=gen, device="cuda").tolist()
    table = torch.full((len(ends), width), -1, dtype=torch.int32)
    for r, js in enumerate(need):
        if js:
            table[r, js[0]:js[-1] + 1] = torch.tensor([spread.pop() for _ in js], dtype=torch.int32)
    return table.cuda(), total


def _quantised(x):
    """x [.., d] -> (codes, scales [..]) of the 8-bit pages."""
    s = x.float().abs().amax(-1).clamp_min(1e-12)
    s = s / torch.full_like(s, 448.0)  # a quotient: torch multiplies by 1 / 448 where the divisor is a Python number
    return (x.float() / s[..., None]).clamp(-448.0, 448.0).to(E4M3), s


def _pool(pages, kv_heads, page, d, dtype, fp8, gen, layers=None):
    shape = (pages, kv_heads, page, d) if layers is None else (layers, pages, kv_heads, page, d)
    x = torch.randn(shape, generator=gen, device="cuda").to(dtype)
    return _quantised(x) if fp8 else (x, None)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    dtype = DTYPES.get(case.get("dtype"), torch.bfloat16)
    kind = case["kind"]
    st = dict(kind=kind)
    if kind == "attend":
        lengths = _lengths(case)
        w = case["window"]
        begins = [max(0, n - w) if w else 0 for n in lengths]
        table, pages = _tables(lengths, begins, case["page"], gen)
        k, ks = _pool(pages, case["kv_heads"], case["page"], case["d"], dtype, case["fp8"], gen)
        v, vs = _pool(pages, case["kv_heads"], case["page"], case["d"], dtype, case["fp8"], gen)
        # queries of twice the keys' size: some tokens get much of the weight, as in a trained model
        q = (randn(case["rows"], case["heads"], case["d"]) * 2).to(dtype)
        st |= dict(q=q, k=k, v=v, ks=ks, vs=vs, table=table, window=w, scale=case["d"] ** -0.5,
                   lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    elif kind == "append":
        count, start = _counts(case)
        table, pages = _tables([s + n for s, n in zip(start, count)], [0] * case["rows"], case["page"], gen)
        k, ks = _pool(pages, case["kv_heads"], case["page"], case["d"], dtype, case["fp8"], gen)
        v, vs = _pool(pages, case["kv_heads"], case["page"], case["d"], dtype, case["fp8"], gen)
        new = lambda: randn(case["rows"], case["tokens"], case["kv_heads"], case["d"]).to(dtype)  # noqa: E731
        st |= dict(new_k=new(), new_v=new(), k=k, v=v, ks=ks, vs=vs, table=table,
                   start=torch.tensor(start, dtype=torch.int32, device="cuda"),
                   count=torch.tensor(count, dtype=torch.int32, device="cuda"))
    elif kind == "copy":
        args = (case["pages"], case["kv_heads"], case["page"], case["d"], dtype, case["fp8"], gen, case["layers"])
        (k, ks), (v, vs) = _pool(*args), _pool(*args)
        order = torch.randperm(case["pages"], generator=gen, device="cuda").tolist()
        n = case["moves"]
        st |= dict(k=k, v=v, ks=ks, vs=vs, src=order[:n], dst=order[n:2 * n])
    elif kind == "gdn":
        rows, hk, hv, slots = case["rows"], case["key_heads"], case["value_heads"], case["slots"]
        C = (2 * hk + hv) * 128
        width = C + hv * 128 + 2 * hv
        width += -width % 128
        at = torch.randperm(slots, generator=gen, device="cuda")[:rows].to(torch.int32)
        if rows > 1:
            at[rows // 2] = -1  # a row of padding
        st |= dict(proj=randn(rows, width).to(dtype), tail=randn(slots, 3, C).to(dtype),
                   conv=(torch.rand(C, 4, generator=gen, device="cuda") - 0.5).to(dtype),
                   A_log=torch.log(1.0 + 15.0 * torch.rand(hv, generator=gen, device="cuda")),
                   dt_bias=(1.0 + 0.1 * randn(hv)).to(dtype), state=randn(slots, hv, 128, 128) * 0.1, at=at, hk=hk,
                   hv=hv, b_off=C + hv * 128, a_off=C + hv * 128 + hv)
    else:
        rows, V, T, N = case["rows"], case["vocab"], case["history"], case["biases"]
        rand = lambda *s: torch.rand(*s, generator=gen, device="cuda")  # noqa: E731
        ints = lambda hi, *s: torch.randint(hi, s, generator=gen, device="cuda", dtype=torch.int32)  # noqa: E731
        past = (rand(rows, T) ** 3 * V).to(torch.int32).clamp_(max=V - 1)  # few tokens often, most seldom
        past = torch.where(torch.arange(T, device="cuda") < 1 + ints(T, rows, 1), past, -1)
        first = ints(V, rows, 1)
        ids = ((first + torch.arange(N, device="cuda") * 7919) % V).to(torch.int32)  # distinct in a row: 7919 is prime
        bits = rand(rows, -(-V // 32) * 32) < case["open"]
        words = (bits.view(rows, -1, 32).long() << torch.arange(32, device="cuda")).sum(-1)
        words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
        st |= dict(logits=(randn(rows, V) * 4).to(dtype), past=past, ids=ids[:, :min(N, V)].contiguous(),
                   values=randn(rows, min(N, V)), mask=words, repetition=1.0 + rand(rows) * 0.3,
                   presence=rand(rows) * 0.5, frequency=rand(rows) * 0.2)
    return st


# --- the plain forms ---------------------------------------------------------------------------------------------
def _gathered(pages, scale, table):
    """The rows' keys or values in order, [rows, kv heads, positions, d] in 32 bits."""
    x = pages[table.long().clamp(min=0)].float()
    if scale is not None:
        x = x * scale[table.long().clamp(min=0)][..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attend(s):
    q, n = s["q"], s["lengths"].long()
    rows, heads, d = q.shape
    k, v = _gathered(s["k"], s["ks"], s["table"]), _gathered(s["v"], s["vs"], s["table"])
    q = q.float().view(rows, k.shape[1], -1, d)
    z = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    at = torch.arange(k.shape[2], device=q.device)
    seen = at < n[:, None]
    if s["window"]:
        seen &= at >= (n - s["window"])[:, None]
    seen = seen[:, None, None]
    z = torch.where(seen, z, -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(z - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0.0, 1.0, total)
    return o.reshape(rows, heads, d).to(s["q"].dtype)


def _plain_append(s):
    T, page = s["new_k"].shape[1], s["k"].shape[2]
    t = torch.arange(T, device="cuda")
    pos = s["start"].long()[:, None] + t
    row, tok = torch.nonzero(t < s["count"].long()[:, None], as_tuple=True)
    pos = pos[row, tok]
    at = s["table"].long()[row, pos // page]
    for_k, for_v = s["new_k"][row, tok], s["new_v"][row, tok]
    if s["ks"] is None:
        s["k"][at, :, pos % page] = for_k
        s["v"][at, :, pos % page] = for_v
        return s["k"], s["v"]
    (ck, sk), (cv, sv) = _quantised(for_k), _quantised(for_v)
    s["k"].view(torch.uint8)[at, :, pos % page] = ck.view(torch.uint8)
    s["v"].view(torch.uint8)[at, :, pos % page] = cv.view(torch.uint8)
    s["ks"][at, :, pos % page] = sk
    s["vs"][at, :, pos % page] = sv
    return s["k"], s["v"], s["ks"], s["vs"]


def _plain_copy(s):
    src, dst = (torch.tensor(x, device="cuda") for x in (s["src"], s["dst"]))
    pools = [s["k"], s["v"]] if s["ks"] is None else [s["k"].view(torch.uint8), s["v"].view(torch.uint8), s["ks"], s["vs"]]
    _ = [p.index_copy_(1, dst, p.index_select(1, src)) for p in pools]
    return [p for p in (s["k"], s["v"], s["ks"], s["vs"]) if p is not None]


def _plain_gdn(s):
    """The step's convolution is rounded to the projection's type, as the chunked form's operands are."""
    hk, hv, proj = s["hk"], s["hv"], s["proj"]
    rows, C = proj.shape[0], s["conv"].shape[0]
    at = s["at"].long()
    live, slot = at >= 0, at.clamp(min=0)
    x = torch.cat([s["tail"][slot], proj[:, None, :C]], 1)
    w = s["conv"].float()
    acc = x[:, 0].float() * w[:, 0]
    acc = acc + x[:, 1].float() * w[:, 1]
    acc = acc + x[:, 2].float() * w[:, 2]
    acc = acc + x[:, 3].float() * w[:, 3]
    y = (acc / (1.0 + torch.exp(-acc))).to(proj.dtype).float()
    q, k, v = y.split((hk * 128, hk * 128, hv * 128), -1)
    q, k, v = q.view(rows, hk, 128), k.view(rows, hk, 128), v.view(rows, hv, 128)
    q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6) * 128 ** -0.5
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    q, k = q.repeat_interleave(hv // hk, 1), k.repeat_interleave(hv // hk, 1)
    b, a = proj[:, s["b_off"]:s["b_off"] + hv].float(), proj[:, s["a_off"]:s["a_off"] + hv].float()
    beta = (1.0 / (1.0 + torch.exp(-b))).to(proj.dtype).float()
    a = a + s["dt_bias"].float()
    g = -torch.exp(s["A_log"]) * torch.where(a > 20.0, a, torch.log1p(torch.exp(a)))
    S = s["state"][slot] * torch.exp(g)[..., None, None]
    u = beta[..., None] * (v - (S * k[..., None]).sum(2))
    S = S + k[..., None] * u[:, :, None]
    o = torch.where(live[:, None, None], (S * q[..., None]).sum(2), 0.0).to(proj.dtype)
    s["state"][slot[live]] = S[live]
    s["tail"][slot[live]] = x[live, 1:]
    return o[:, :, None], s["state"], s["tail"]


def _plain_constrain(s):
    z = s["logits"].float()
    rows, V = z.shape
    past = s["past"].long()
    n = torch.zeros_like(z).scatter_add_(1, past.clamp(min=0), (past >= 0).float())
    r = s["repetition"][:, None]
    penal = torch.where(z > 0, z / r, z * r) - (s["frequency"][:, None] * n + s["presence"][:, None])
    z = torch.where(n > 0, penal, z)
    z = z + torch.zeros_like(z).scatter_add_(1, s["ids"].long(), s["values"])
    at = torch.arange(V, device=z.device)
    seen = (s["mask"][:, at // 32] >> (at % 32)) & 1
    return torch.where(seen != 0, z, -math.inf)


def run(state):
    s = state
    kind = s["kind"]
    if not own:
        return {"attend": _plain_attend, "append": _plain_append, "copy": _plain_copy, "gdn": _plain_gdn,
                "constrain": _plain_constrain}[kind](s)
    if own:
        from basal_b200 import ops
        if kind == "attend":
            return ops.paged_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["scale"], s["window"],
                                       s["ks"], s["vs"])
        if kind == "append":
            ops.kv_append(s["new_k"], s["new_v"], s["k"], s["v"], s["table"], s["start"], s["count"], s["ks"], s["vs"])
            return (s["k"], s["v"]) if s["ks"] is None else (s["k"], s["v"], s["ks"], s["vs"])
        if kind == "copy":
            pools = [p for p in (s["k"], s["v"], s["ks"], s["vs"]) if p is not None]
            ops.kv_copy_pages(pools, s["src"], s["dst"])
            return pools
        if kind == "gdn":
            o = ops.gdn_step(s["proj"], s["tail"], s["conv"], s["A_log"], s["dt_bias"], s["state"], s["hk"], s["hv"],
                             s["b_off"], s["a_off"], s["at"])
            return o, s["state"], s["tail"]
        return ops.constrain_logits(s["logits"], s["mask"], s["past"], s["repetition"], s["presence"], s["frequency"],
                                    s["ids"], s["values"])


def work(case):
    kind = case["kind"]
    size = 4 if case.get("dtype") == "fp32" else 2
    if kind in ("attend", "append", "copy"):
        token = case["kv_heads"] * (case["d"] + 4 if case["fp8"] else case["d"] * 2) * 2  # its key and value in a page
    if kind == "attend":
        n = sum(min(x, case["window"]) if case["window"] else x for x in _lengths(case))
        io = case["rows"] * case["heads"] * case["d"] * 2 * 2
        return dict(bytes=n * token + io + 4 * n // case["page"], flops=4 * n * case["heads"] * case["d"])
    if kind == "append":
        n = sum(_counts(case)[0])
        return dict(bytes=n * (token + case["kv_heads"] * case["d"] * 2 * 2), flops=n * case["kv_heads"] * case["d"] * 4)
    if kind == "copy":
        return dict(bytes=2 * case["layers"] * case["moves"] * case["page"] * token, flops=0)
    if kind == "gdn":
        n, hk, hv = max(1, case["rows"] - 1), case["key_heads"], case["value_heads"]
        C = (2 * hk + hv) * 128
        states, rest = n * hv * 128 * 128 * 4 * 2, n * (C * (1 + 3 + 3) + hv * 128 + 2 * hv) * 2 + C * 8
        return dict(bytes=states + rest, flops=n * hv * 128 * 128 * 7)
    n = case["rows"] * case["vocab"]
    # a logit is needed where the mask leaves its token; half the history's places are taken
    words = 1.0 - (1.0 - case["open"]) ** (32 // size)  # 32-byte sectors that hold such a logit
    return dict(bytes=n * 4 + n / 8 + n * size * (words if case["open"] < 1 else 1) +
                case["rows"] * (case["history"] * 2 + case["biases"] * 8), flops=n * 4)


def exact(case, seed):
    """The outputs from the definitions, in 64 bits."""
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "attend":
        q, table = s["q"].double(), s["table"].long()
        rows, heads, d = q.shape
        per, page = heads // s["k"].shape[1], s["k"].shape[2]
        o = torch.zeros_like(q)
        for r, n in enumerate(s["lengths"].tolist()):
            first = max(0, n - s["window"]) if s["window"] else 0
            if n == 0:
                continue
            at = torch.arange(first, n, device="cuda")
            where, inside = table[r, torch.div(at, page, rounding_mode="floor")], at.remainder(page)
            for h in range(s["k"].shape[1]):
                k, v = s["k"][where, h, inside].double(), s["v"][where, h, inside].double()
                if s["ks"] is not None:
                    k, v = k * s["ks"][where, h, inside, None], v * s["vs"][where, h, inside, None]
                p = torch.softmax(q[r, h * per:(h + 1) * per] @ k.T / math.sqrt(d), -1)
                o[r, h * per:(h + 1) * per] = p @ v
        return o
    if kind == "append":
        count, start = _counts(case)
        got = [x.double() for x in (s["k"], s["v"], s["ks"], s["vs"]) if x is not None]
        page, table = case["page"], s["table"].tolist()
        for r in range(case["rows"]):
            at = torch.arange(start[r], start[r] + count[r], device="cuda")
            where, inside = s["table"][r].long()[at // page], at % page
            for i, name in enumerate(("new_k", "new_v")):
                x = s[name][r, :count[r]].double()
                if s["ks"] is not None:
                    top = x.abs().amax(-1).clamp_min(1e-12) / 448.0
                    # the scale is held in 32 bits, and a code stands for the value over that scale
                    got[2 + i][where, :, inside] = top
                    x = (x / top.float().double()[..., None]).float().to(E4M3).double()
                got[i][where, :, inside] = x
        # the pages' own type: 8-bit codes as the values they stand for
        return [x.float() for x in got]
    if kind == "copy":
        got = [x.clone() for x in (s["k"], s["v"], s["ks"], s["vs"]) if x is not None]
        for x, y in zip(got, (x for x in (s["k"], s["v"], s["ks"], s["vs"]) if x is not None)):
            for a, b in zip(s["src"], s["dst"]):
                x[:, b] = y[:, a]
        return got
    if kind == "gdn":
        hk, hv, proj, C = s["hk"], s["hv"], s["proj"], s["conv"].shape[0]
        o = torch.zeros(proj.shape[0], hv, 1, 128, dtype=torch.float64, device="cuda")
        state, tail = s["state"].double(), s["tail"].double()
        rep = hv // hk
        for r, slot in enumerate(s["at"].tolist()):
            if slot < 0:
                continue
            window = torch.cat([tail[slot], proj[r:r + 1, :C].double()])
            y = torch.einsum("tc,ct->c", window, s["conv"].double())
            y = (y * torch.sigmoid(y)).to(proj.dtype).double()
            q, k = y[:hk * 128].view(hk, 128), y[hk * 128:2 * hk * 128].view(hk, 128)
            v = y[2 * hk * 128:].view(hk, rep, 128)
            q = q / torch.sqrt(q.square().sum(-1, keepdim=True) + 1e-6) / math.sqrt(128.0)
            k = k / torch.sqrt(k.square().sum(-1, keepdim=True) + 1e-6)
            beta = torch.sigmoid(proj[r, s["b_off"]:s["b_off"] + hv].double()).to(proj.dtype).double().view(hk, rep)
            a = proj[r, s["a_off"]:s["a_off"] + hv].double() + s["dt_bias"].double()
            decay = torch.exp(-torch.exp(s["A_log"].double()) * torch.nn.functional.softplus(a, threshold=1e9))
            S = state[slot].view(hk, rep, 128, 128) * decay.view(hk, rep, 1, 1)
            u = beta[..., None] * (v - torch.einsum("hrkv,hk->hrv", S, k))
            S = S + torch.einsum("hk,hrv->hrkv", k, u)
            o[r, :, 0] = torch.einsum("hrkv,hk->hrv", S, q).reshape(hv, 128)
            state[slot] = S.reshape(hv, 128, 128)
            tail[slot] = window[1:]
        return o, state, tail
    got = torch.full(s["logits"].shape, -math.inf, dtype=torch.float64, device="cuda")
    V = case["vocab"]
    for r in range(case["rows"]):
        z = s["logits"][r].double()
        past = s["past"][r]
        n = torch.bincount(past[past >= 0].long(), minlength=V).double()
        lower = torch.minimum(z * s["repetition"][r].double(), z / s["repetition"][r].double())
        z = torch.where(n > 0, lower - s["presence"][r].double() - n * s["frequency"][r].double(), z)
        z[s["ids"][r].long()] += s["values"][r].double()
        left = (s["mask"][r][:, None] >> torch.arange(32, device="cuda") & 1).flatten()[:V] != 0
        got[r, left] = z[left]
    return got
