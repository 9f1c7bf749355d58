"""The paged key / value cache on the GPU: basal::paged_attention, basal::kv_append, basal::kv_copy_pages.

Attention against the same sums in 64 bits. Its tolerance, per value: the output's rounding, eps / 2 of the value, plus
the work in 32 bits: with a = sum_t p_t |v_t|, a weight p_t is off by the relative error of exp(z): that of z's sum of D
products, (D + 8) 2^-24 scale sum_d |q_d k_td|, of its scaling and of the exponential, |z| 2^-22 + 2^-20; twice that
for the quotient (numerator and sum); 2^-17 for weights split into two 16-bit halves (2^-11, fp16's half step, for
8-bit pages under bf16 queries, whose output is rounded by 2^-8); and the sums over the row's
positions, 2^-23 for each of n / 16 + 64 additions. Every position that no row may read holds NaN in the pools.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, FP16, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from basal_b200 import _lib, ops
    _lib.device_faults(0)
    yield ops
    assert _lib.device_faults(0) == 0


def faults():
    from basal_b200 import _lib
    return _lib.device_faults(0)


def quantised(x):
    s = x.float().abs().amax(-1).clamp_min(1e-12)
    s = s / torch.full_like(s, 448.0)
    return (x.float() / s[..., None]).clamp(-448, 448).to(E4M3), s


class Pool:
    """A cache of rows with the given lengths, spread over random pages; whatever no row holds is NaN."""

    def __init__(self, lengths, Hk, D, ps, dtype, fp8, window=0, seed=0, spare=3, order="head"):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        need = [range(max(0, n - window) // ps if window else 0, -(-n // ps)) for n in lengths]
        N = sum(map(len, need)) + spare
        ids = torch.randperm(N, generator=g, device="cuda").tolist()
        width = max(1, max(-(-n // ps) for n in lengths))
        table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        live = torch.zeros(N, ps, dtype=torch.bool)
        for r, (n, js) in enumerate(zip(lengths, need)):
            for j in js:
                table[r, j] = ids.pop()
                lo = max(0, n - window) if window else 0
                at = torch.arange(ps) + j * ps
                live[table[r, j]] = (at < n) & (at >= lo)
        self.table, live = table.cuda(), live.cuda()
        self.full = [torch.randn(N, Hk, ps, D, device="cuda", generator=g).to(dtype) for _ in range(2)]
        self.scales = [None, None]
        if fp8:
            (k, ks), (v, vs) = map(quantised, self.full)
            dead = ~live[:, None, :].expand(N, Hk, ps)
            self.scales = [s.masked_fill(dead, float("nan")) for s in (ks, vs)]
            self.full = [c.view(torch.uint8).masked_fill(dead[..., None], 0x7F).view(E4M3) for c in (k, v)]
        else:
            self.full = [x.masked_fill(~live[:, None, :, None], float("nan")) for x in self.full]
        if order == "token":  # [pages, page size, heads, D] behind the same shape
            self.full = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in self.full]
        elif order == "layer":  # one layer of several
            many = [torch.zeros(x.shape[0], 3, *x.shape[1:], dtype=x.dtype, device="cuda") for x in self.full]
            for m, x in zip(many, self.full):
                m.view(torch.uint8)[:, 1] = x.contiguous().view(torch.uint8)
            self.full = [m[:, 1] for m in many]
        self.window, self.ps = window, ps

    def row(self, r):
        """The row's keys and values in 64 bits, [Hk, positions, D]."""
        n = int(self.lengths[r])
        at = torch.arange(max(0, n - self.window) if self.window else 0, n, device="cuda")
        page, off = self.table[r].long()[at // self.ps], at % self.ps
        out = []
        for x, s in zip(self.full, self.scales):
            y = x.view(torch.uint8)[page, :, off].view(x.dtype) if s is not None else x[page, :, off]
            y = y.double()
            out.append((y if s is None else y * s[page, :, off].double()[..., None]).transpose(0, 1))
        return out


def check(ops, pool, q, scale, got):
    rows, H, D = q.shape
    fi = torch.finfo(q.dtype)
    weight = 2.0 ** -11 if pool.scales[0] is not None and q.dtype == BF else 2.0 ** -17
    for r in range(rows):
        k, v = pool.row(r)
        Hk, n = k.shape[:2]
        if n == 0:
            assert torch.equal(got[r], torch.zeros_like(got[r]))
            continue
        qr = q[r].double().view(Hk, H // Hk, D)
        z = qr @ k.transpose(1, 2) * scale
        p = torch.softmax(z, -1)
        o, a = p @ v, p @ v.abs()
        size = scale * (qr.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True)
        ez = (D + 8) * 2.0 ** -24 * size + z.abs().amax(-1, keepdim=True) * 2.0 ** -22 + 2.0 ** -20
        # a value below the type's smallest normal one is rounded to a multiple of tiny * eps: off by half of that
        tol = fi.eps / 2 * o.abs().clamp(min=fi.tiny) + a * (2 * ez + weight + (n / 16 + 64) * 2.0 ** -23)
        off = (got[r].double().view_as(o) - o).abs()
        assert torch.isfinite(got[r]).all(), r
        assert (off <= tol).all(), (r, n, (off / tol).max().item())


def attend(ops, pool, q, scale):
    return ops.paged_attention(q, *pool.full, pool.table, pool.lengths, scale, pool.window, *pool.scales)


EDGES = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 100, 255, 256, 257, 300, 511, 513, 1000]


@pytest.mark.parametrize("dtype, fp8", [(BF, False), (FP16, False), (BF, True), (FP16, True)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H, Hk, ps", [(16, 4, 64), (5, 5, 16), (6, 2, 24), (8, 1, 1), (24, 2, 128), (34, 2, 5)])
def test_attention(ops, dtype, fp8, D, H, Hk, ps):
    pool = Pool(EDGES, Hk, D, ps, dtype, fp8, seed=D + H)
    q = torch.randn(len(EDGES), H, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(H)) * 2
    q = q.to(dtype)
    check(ops, pool, q, D ** -0.5, attend(ops, pool, q, D ** -0.5))


@pytest.mark.parametrize("window", [1, 7, 16, 100, 300, 5000])
@pytest.mark.parametrize("fp8, ps", [(False, 64), (True, 24), (False, 16)])
def test_attention_window(ops, window, fp8, ps):
    """Pages before the window are not in the table (-1) and are not read."""
    lengths = [0, 1, 15, 16, 17, 100, 130, 600, 2049, 4111]
    pool = Pool(lengths, 2, 128, ps, BF, fp8, window, seed=window)
    q = (torch.randn(len(lengths), 8, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) * 2)
    check(ops, pool, q.to(BF), 128 ** -0.5, attend(ops, pool, q.to(BF), 128 ** -0.5))


@pytest.mark.parametrize("D, H, Hk, fp8", [(128, 16, 4, False), (128, 8, 8, True), (64, 12, 1, False),
                                           (256, 4, 2, False)])
def test_attention_long(ops, D, H, Hk, fp8):
    lengths = [30001, 5, 70000, 4096]
    pool = Pool(lengths, Hk, D, 64, BF, fp8, seed=5)
    q = (torch.randn(4, H, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)) * 2).to(BF)
    check(ops, pool, q, D ** -0.5, attend(ops, pool, q, D ** -0.5))


@pytest.mark.parametrize("order", ["token", "layer"])
@pytest.mark.parametrize("fp8", [False, True])
def test_attention_strided_pages_and_queries(ops, order, fp8):
    pool = Pool(EDGES, 4, 128, 16, BF, fp8, seed=3, order=order)
    g = torch.Generator(device="cuda").manual_seed(4)
    wide = torch.randn(len(EDGES), 8, 256, device="cuda", generator=g).to(BF)
    for q in (wide[..., :128], wide[..., 3:131]):  # a strided view, and one that is not aligned
        check(ops, pool, q, 0.1, attend(ops, pool, q, 0.1))
        assert torch.equal(attend(ops, pool, q, 0.1), attend(ops, pool, q.contiguous(), 0.1))


@pytest.mark.parametrize("fp8", [False, True])
def test_attention_extreme_logits(ops, fp8):
    """One key far above the others, all keys equal, all logits far below zero, and weights that underflow."""
    pool = Pool([700] * 4, 2, 128, 64, BF, fp8, seed=8)
    q = torch.randn(4, 8, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9)).to(BF)
    q[0] *= 100
    q[1] = 0
    k, _ = pool.row(2)
    q[2] = (-40 * k[0, 0]).to(BF)
    q[3] *= 1e-30
    check(ops, pool, q, 128 ** -0.5, attend(ops, pool, q, 128 ** -0.5))


def test_attention_8bit_scales_of_all_sizes(ops):
    """Scales from 1e-30 to 1e30 within a row: values are code * scale in 32 bits whatever the other tokens' scales."""
    pool = Pool([333, 40], 2, 128, 16, BF, True, seed=11)
    g = torch.Generator(device="cuda").manual_seed(12)
    pool.scales[1] = pool.scales[1] * 10.0 ** (torch.rand(pool.scales[1].shape, device="cuda", generator=g) * 60 - 30)
    q = torch.randn(2, 4, 128, device="cuda", generator=g).to(BF)
    check(ops, pool, q, 128 ** -0.5, attend(ops, pool, q, 128 ** -0.5))


@pytest.mark.parametrize("fp8", [False, True])
def test_attention_row_alone_and_among_others(ops, fp8):
    lengths = [5000, 1, 300, 0, 20000, 257]
    pool = Pool(lengths, 4, 128, 64, BF, fp8, seed=6)
    q = torch.randn(6, 16, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7)).to(BF)
    whole = attend(ops, pool, q, 0.09)
    for r in range(6):
        alone = ops.paged_attention(q[r:r + 1], *pool.full, pool.table[r:r + 1], pool.lengths[r:r + 1], 0.09, 0,
                                    *pool.scales)
        assert torch.equal(alone[0], whole[r]), r
    assert torch.equal(attend(ops, pool, q, 0.09), whole)


def test_attention_infinite_and_nan_tokens(ops):
    """A NaN in a token that a row reads reaches that row's heads of that key head, and no other row."""
    pool = Pool([100, 100], 2, 128, 16, BF, False, seed=13)
    q = torch.randn(2, 4, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(14)).to(BF)
    clean = attend(ops, pool, q, 0.09)
    pool.full[0][pool.table[0, 2].long(), 1, 3, 5] = float("nan")
    got = attend(ops, pool, q, 0.09)
    assert got[0, 2:].isnan().all() and torch.equal(got[0, :2], clean[0, :2]) and torch.equal(got[1], clean[1])


def test_attention_bad_pages_and_lengths(ops):
    """A page that is not there, or a length past the table: a NaN row and the fault bit, the other rows unharmed."""
    from basal_b200 import _lib  # noqa: F401
    pool = Pool([300, 300, 300, 40], 2, 128, 16, BF, False, seed=15)
    q = torch.randn(4, 4, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(16)).to(BF)
    clean = attend(ops, pool, q, 0.09)
    pool.table[0, 7] = -1
    pool.table[1, 18] = pool.full[0].shape[0]
    got = attend(ops, pool, q, 0.09)
    assert faults() == 64
    assert got[:2].isnan().all() and torch.equal(got[2:], clean[2:])
    pool.lengths[2] = pool.table.shape[1] * 16 + 1
    pool.lengths[3] = -5
    got = attend(ops, pool, q, 0.09)
    assert faults() == 64
    assert got[2].isnan().all() and torch.equal(got[3], torch.zeros_like(got[3]))


def test_attention_far_pages(ops):
    """Pages whose elements lie past 2^31: 64-bit offsets (keys and values of one pool of 4.5 GB each)."""
    Hk, D, ps = 2, 128, 64
    N = (1 << 31) // (Hk * D * ps) + 200
    pools = [torch.empty(N, Hk, ps, D, dtype=BF, device="cuda") for _ in range(2)]
    small = Pool([500, 77], Hk, D, ps, BF, False, seed=17)
    at = N - 1 - torch.arange(small.full[0].shape[0], device="cuda")
    for big, x in zip(pools, small.full):
        big[at] = x
    q = torch.randn(2, 8, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(18)).to(BF)
    far = torch.where(small.table >= 0, N - 1 - small.table, -1)
    got = ops.paged_attention(q, *pools, far, small.lengths, 0.09)
    assert torch.equal(got, attend(ops, small, q, 0.09))
    new = torch.randn(2, 1, Hk, D, device="cuda").to(BF)
    ops.kv_append(new, new, *pools, far, small.lengths - 1)
    assert torch.equal(pools[1][far[0, 7].long(), :, 499 % ps], new[0, 0])
    ops.kv_copy_pages([p[None] for p in pools], [N - 1], [N - 150])
    assert torch.equal(pools[0][N - 1].view(torch.int16), pools[0][N - 150].view(torch.int16))


def test_attention_captured_and_on_another_stream(ops):
    """Two graphs that share a memory pool, replayed in turn on lengths and tables that changed, and a side stream."""
    pool = Pool([9000, 300], 4, 128, 64, BF, False, seed=19)
    q = torch.randn(2, 16, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(20)).to(BF)
    want = attend(ops, pool, q, 0.09)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(attend(ops, pool, q, 0.09))
        graphs.append(g)
    graphs[0].replay()
    assert torch.equal(outs[0], want)
    pool.lengths[0] = 4000
    short = attend(ops, pool, q, 0.09)
    graphs[1].replay()
    assert torch.equal(outs[1], short) and not torch.equal(short, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attend(ops, pool, q, 0.09)
    side.synchronize()
    assert torch.equal(got, short)


def test_attention_no_rows_and_no_pages(ops):
    k = torch.zeros(0, 2, 16, 64, dtype=BF, device="cuda")
    table = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    z = torch.zeros(3, dtype=torch.int32, device="cuda")
    q = torch.ones(3, 4, 64, dtype=BF, device="cuda")
    assert torch.equal(ops.paged_attention(q, k, k, table, z, 1.0), torch.zeros_like(q))
    assert ops.paged_attention(q[:0], k, k, table[:0], z[:0], 1.0).shape == (0, 4, 64)


def refused(f, *a):
    with pytest.raises(ValueError):
        f(*a)


def test_refusals(ops):
    k = torch.zeros(4, 2, 16, 64, dtype=BF, device="cuda")
    t, n = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    q = torch.ones(1, 4, 64, dtype=BF, device="cuda")
    refused(ops.paged_attention, q.float(), k, k, t, n, 1.0)                       # 32-bit queries
    refused(ops.paged_attention, q.half(), k, k, t, n, 1.0)                        # another type than the pages
    refused(ops.paged_attention, q[:, :3], k, k, t, n, 1.0)                        # heads that do not share evenly
    refused(ops.paged_attention, q[..., :32], k[..., :32], k[..., :32], t, n, 1.0)  # heads of 32
    refused(ops.paged_attention, q, k, k, t.long(), n, 1.0)                        # 64-bit tables
    refused(ops.paged_attention, q, k, k, t, n.long(), 1.0)
    refused(ops.paged_attention, q, k, k, t[:0], n, 1.0)                           # a table of other rows
    refused(ops.paged_attention, q, k, k[:, :1], t, n, 1.0)
    refused(ops.paged_attention, q, k, k, t, n, 1.0, -1)                           # a negative window
    refused(ops.paged_attention, q, k.to(E4M3), k.to(E4M3), t, n, 1.0)             # 8-bit pages without scales
    refused(ops.paged_attention, q, k, k, t, n, 1.0, 0, k[..., 0].float(), k[..., 0].float())
    refused(ops.paged_attention, q, k.cpu(), k.cpu(), t, n, 1.0)
    odd = torch.zeros(4, 2, 16, 68, dtype=BF, device="cuda")[..., :64]             # rows not 16-byte aligned
    refused(ops.paged_attention, q, odd, odd, t, n, 1.0)
    x = torch.ones(1, 3, 2, 64, dtype=BF, device="cuda")
    refused(ops.kv_append, x.float(), x.float(), k, k, t, n)
    refused(ops.kv_append, x.half(), x.half(), k, k, t, n)
    refused(ops.kv_append, x[:, :, :1], x[:, :, :1], k, k, t, n)
    refused(ops.kv_append, x, x[:, :2], k, k, t, n)
    refused(ops.kv_append, x, x, k, k, t, n.long())
    refused(ops.kv_append, x, x, k, k, t, n, n.float())
    p = torch.zeros(2, 6, 8, dtype=torch.int32, device="cuda")
    refused(ops.kv_copy_pages, [p], [0], [1, 2])
    refused(ops.kv_copy_pages, [p], [0], [6])
    refused(ops.kv_copy_pages, [p], [-1], [2])
    refused(ops.kv_copy_pages, [p], [0, 1], [2, 2])      # a page written twice
    refused(ops.kv_copy_pages, [p], [0, 1], [1, 2])      # a page both read and written
    refused(ops.kv_copy_pages, [p], [3], [3])
    refused(ops.kv_copy_pages, [p, p[:, :5]], [0], [1])
    refused(ops.kv_copy_pages, [p.transpose(0, 2)], [0], [1])
    refused(ops.kv_copy_pages, [torch.zeros(2, 6, 3, dtype=torch.uint8, device="cuda")], [0], [1])  # pages of 3 bytes
    assert not p.any()


# --- append ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype, fp8", [(BF, False), (FP16, False), (BF, True), (FP16, True)])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T, Hk, ps", [(1, 4, 64), (37, 1, 24), (130, 2, 16), (3, 3, 1)])
def test_append(ops, dtype, fp8, D, T, Hk, ps):
    """Every position as the plain indexing leaves it, bit for bit, the others (and the pages of no row) untouched."""
    g = torch.Generator(device="cuda").manual_seed(T + D)
    start = [0, 5, -1, 63, 64, 17]
    count = [T, 1, T, max(0, T - 2), T + 9, 0]
    rows = len(start)
    lengths = [max(s, 0) + T for s in start]
    pool = Pool(lengths, Hk, D, ps, dtype, fp8, seed=T)
    k, v = (torch.randn(rows, T, Hk, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    k[0, 0, 0] = 0                       # an all-zero token
    k[3 % rows, 0, 0, 0] = 1000.0        # an outlier
    raw = lambda x: x.view(torch.uint8 if fp8 else torch.int16)  # noqa: E731
    want = [raw(x).clone() for x in pool.full]
    wants = [None if s is None else s.view(torch.int32).clone() for s in pool.scales]
    for i, x in enumerate((k, v)):
        codes, s = quantised(x) if fp8 else (x, None)
        for r in range(rows):
            for t in range(min(T, count[r]) if start[r] >= 0 else 0):
                pos = start[r] + t
                page = int(pool.table[r, pos // ps])
                want[i][page, :, pos % ps] = raw(codes)[r, t]
                if fp8:
                    wants[i][page, :, pos % ps] = s.view(torch.int32)[r, t]
    args = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (start, count)]
    ops.kv_append(k, v, *pool.full, pool.table, *args, *pool.scales)
    for x, w in zip(pool.full, want):
        assert torch.equal(raw(x), w)
    for s, w in zip(pool.scales, wants):
        assert s is None or torch.equal(s.view(torch.int32), w)


def test_append_8bit_equals_the_activation_quantiser(ops):
    pool = Pool([640], 3, 128, 64, BF, True, seed=21)
    x = torch.randn(1, 640, 3, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(22)).to(BF)
    ops.kv_append(x, x, *pool.full, pool.table, torch.zeros(1, dtype=torch.int32, device="cuda"), None, *pool.scales)
    q, s = ops.fp8_act_quant(x.view(-1, 128))
    at = pool.table[0].long()
    got = pool.full[0].view(torch.uint8)[at].transpose(1, 2).reshape(-1, 128)
    assert torch.equal(got, q.view(torch.uint8))
    assert torch.equal(pool.scales[0][at].transpose(1, 2).reshape(-1), s.view(-1))


@pytest.mark.parametrize("dtype, size", [(FP16, 2e-7), (FP16, 60000.0), (BF, 1e-39), (BF, 1e38), (BF, 1e-13)])
def test_append_8bit_of_tiny_and_huge_tokens(ops, dtype, size):
    """Tokens of the type's smallest and largest values (subnormal ones among them) take the quantiser's codes and scales."""
    pool = Pool([64], 2, 128, 16, dtype, True, seed=27)
    x = torch.randn(1, 64, 2, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(28)).clamp(-1, 1)
    x = (x.double() * size).to(dtype)
    ops.kv_append(x, x, *pool.full, pool.table, torch.zeros(1, dtype=torch.int32, device="cuda"), None, *pool.scales)
    q, s = ops.fp8_act_quant(x.view(-1, 128))
    at = pool.table[0].long()
    assert torch.equal(pool.full[0].view(torch.uint8)[at].transpose(1, 2).reshape(-1, 128), q.view(torch.uint8))
    assert torch.equal(pool.scales[1][at].transpose(1, 2).reshape(-1), s.view(-1))


def test_append_strided_sources_without_count(ops):
    """[rows, heads, tokens, D] seen as [rows, tokens, heads, D], a slice of a wider projection, and unaligned ones."""
    for fp8 in (False, True):
        a, b, c = (Pool([50, 50], 2, 128, 16, BF, fp8, seed=23) for _ in range(3))
        g = torch.Generator(device="cuda").manual_seed(24)
        wide = torch.randn(2, 2, 9, 140, device="cuda", generator=g).to(BF)
        start = torch.tensor([40, 7], dtype=torch.int32, device="cuda")
        x, y = wide[..., :128].transpose(1, 2), wide[..., 3:131].transpose(1, 2)
        ops.kv_append(x, y, *a.full, a.table, start, None, *a.scales)
        ops.kv_append(x.contiguous(), y.contiguous(), *b.full, b.table, start, None, *b.scales)
        view = torch.zeros(2, 9, 2, 256, dtype=BF, device="cuda")
        view[..., :128] = x
        ops.kv_append(view[..., :128], y, *c.full, c.table, start, None, *c.scales)
        for p, q, r in zip(a.full, b.full, c.full):
            assert torch.equal(p.view(torch.uint8), q.view(torch.uint8))
            assert torch.equal(p.view(torch.uint8), r.view(torch.uint8))


def test_append_nan_and_inf_tokens(ops):
    """A token's NaN or infinity marks its scale and nobody else's."""
    pool = Pool([4], 1, 128, 16, BF, True, seed=25)
    x = torch.ones(1, 4, 1, 128, dtype=BF, device="cuda")
    x[0, 1, 0, 5], x[0, 2, 0, 6] = float("nan"), float("inf")
    ops.kv_append(x, x, *pool.full, pool.table, torch.zeros(1, dtype=torch.int32, device="cuda"), None, *pool.scales)
    s = pool.scales[0][pool.table[0, 0].long(), 0, :4]
    assert torch.isfinite(s[[0, 3]]).all() and s[1].isnan() and s[2].isinf()


def test_append_where_no_page_is(ops):
    pool = Pool([40, 40], 2, 64, 16, BF, False, seed=26)
    before = [x.clone().view(torch.int16) for x in pool.full]
    x = torch.ones(2, 4, 2, 64, dtype=BF, device="cuda")
    pool.table[0, 1] = 10 ** 6
    pool.table[1, 2] = -1
    # row 0: positions 14, 15 fit, 16, 17 do not; row 1: past the table
    ops.kv_append(x, x, *pool.full, pool.table, torch.tensor([14, 46], dtype=torch.int32, device="cuda"))
    assert faults() == 64
    at = pool.table[0, 0].long()
    for b, p in zip(before, pool.full):
        p = p.view(torch.int16)
        changed = (p != b).nonzero()
        assert set(changed[:, 0].tolist()) == {int(at)} and set(changed[:, 2].tolist()) == {14, 15}
    ops.kv_append(x, x, *pool.full, pool.table, torch.tensor([-1, 2 ** 31 - 1], dtype=torch.int32, device="cuda"))
    assert faults() == 64


# --- copies ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("moves", [1, 3, 32, 33, 1500, 2500])
@pytest.mark.parametrize("fp8", [False, True])
def test_copy_pages(ops, moves, fp8):
    N, g = 2 * moves + 5, torch.Generator(device="cuda").manual_seed(moves)
    pools = [torch.randint(0, 255, (2, N, 1, 4, 64), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
    pools.append(torch.randn(3, N, 1, 3, generator=g, device="cuda"))  # pages of 12 bytes: no 16-byte rows
    if fp8:
        pools[0] = pools[0].view(E4M3)
    order = torch.randperm(N, generator=g, device="cuda").tolist()
    src, dst = order[:moves], order[moves:2 * moves]
    raw = [p.view(torch.uint8) for p in pools]
    want = [r.clone() for r in raw]
    for w, r in zip(want, raw):
        w[:, dst] = r[:, src]
    ops.kv_copy_pages(pools, src, dst)
    for w, r in zip(want, raw):
        assert torch.equal(w, r)
    ops.kv_copy_pages(pools, [], [])
    ops.kv_copy_pages([], src, dst)
    for w, r in zip(want, raw):
        assert torch.equal(w, r)


def test_a_page_copied_to_many(ops):
    p = torch.arange(2 * 40 * 16, dtype=torch.int32, device="cuda").view(2, 40, 16)
    ops.kv_copy_pages([p], [7] * 35, list(range(5)) + list(range(10, 40)))
    assert torch.equal(p[:, list(range(5)) + list(range(10, 40))], p[:, 7:8].expand(2, 35, 16))


def test_copy_and_append_captured(ops):
    """A captured copy keeps its own list of moves: the host's lists may be gone or changed before the replay."""
    p = torch.arange(6 * 16, dtype=torch.int32, device="cuda").view(1, 6, 16)
    src, dst = [0, 1], [4, 5]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv_copy_pages([p], src, dst)
    src[0], dst[1] = 3, 3
    p[0, 0] = -1
    g.replay()
    assert torch.equal(p[0, 4], p[0, 0]) and torch.equal(p[0, 5], p[0, 1]) and int(p[0, 3, 0]) == 48


# --- inputs that are contiguous and not aligned --------------------------------------------------------------------
@pytest.mark.parametrize("offset", [1, 3, 4, 8])
@pytest.mark.parametrize("fp8", [False, True])
def test_one_row_at_any_offset(ops, fp8, offset):
    """One row's query, key and value as slices of a projection at any column: contiguous views, most not 16-byte
    aligned, one with a row stride that is no multiple of 8."""
    pool, same = (Pool([70], 2, 128, 16, BF, fp8, seed=29) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(30)
    proj = torch.randn(1, offset + 8 * 128 + 3, device="cuda", generator=g).to(BF)
    q = proj[:, offset:offset + 512].view(1, 4, 128)
    k, v = (proj[:, offset + at:offset + at + 256].view(1, 1, 2, 128) for at in (512, 768))
    assert q.is_contiguous() and k.is_contiguous()
    start = torch.tensor([69], dtype=torch.int32, device="cuda")
    ops.kv_append(k, v, *pool.full, pool.table, start, None, *pool.scales)
    ops.kv_append(k.clone(), v.clone(), *same.full, same.table, start, None, *same.scales)
    for a, b in zip(pool.full, same.full):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(attend(ops, pool, q, 0.09), attend(ops, same, q.clone(), 0.09))


# --- 8-bit values under weights of any size ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, FP16])
@pytest.mark.parametrize("n", [300, 6000])
@pytest.mark.parametrize("ratio", [16, 20, 24, 40, 80, 100])
def test_attention_8bit_large_scale_of_an_unlikely_token(ops, dtype, n, ratio):
    """A token whose value scale is 2^ratio times the others' and whose logit is 60 below theirs (a weight of 2^-86): what
    counts is the product of scale and weight, from nothing (2^16) to nearly all (2^100) of the output."""
    pool = Pool([n, 40], 2, 128, 16, dtype, True, seed=32)
    g = torch.Generator(device="cuda").manual_seed(33)
    one = torch.randn(2, 2, 1, 128, device="cuda", generator=g).expand(2, 2, 2, 128) * 2  # a key head's queries alike
    q = (one * torch.tensor([1.0, 0.9], device="cuda")[:, None]).reshape(2, 4, 128).to(dtype)
    for r, at in ((0, n // 2 + 3), (0, 5), (1, 17)):
        page, off = pool.table[r, at // 16].long(), at % 16
        x = one[r, :, 0]
        codes, s = quantised(x * (-60 / (128 ** -0.5 * x.square().sum(-1, keepdim=True))))
        pool.full[0].view(torch.uint8)[page, :, off] = codes.view(torch.uint8)
        pool.scales[0][page, :, off] = s
        pool.scales[1][page, :, off] *= 2.0 ** ratio
    got = attend(ops, pool, q, 128 ** -0.5)
    if dtype == BF or ratio < 100:
        return check(ops, pool, q, 128 ** -0.5, got)
    # 2^100 e^-60 is 2^13.4 (2^22 for the queries of 0.9), and values reach 4: past fp16's largest value, 65504, whose rounding
    # is an infinity; the others are compared to 2^-6, well above check()'s bound for them
    for r in range(2):
        k, v = pool.row(r)
        p = torch.softmax(q[r].double().view(2, 2, 128) @ k.transpose(1, 2) * 128 ** -0.5, -1)
        o, a = (p @ v).view(4, 128), (p @ v.abs()).view(4, 128)
        y = got[r].double()
        large, small = o.abs() > 65520 + 2.0 ** -6 * a, o.abs() < 65504 - 2.0 ** -6 * a
        assert (y[large] == o[large].sign() * float("inf")).all()
        assert ((y - o).abs() <= 2.0 ** -6 * a)[small].all()


@pytest.mark.parametrize("dtype, fp8", [(BF, False), (FP16, False), (BF, True), (FP16, True)])
@pytest.mark.parametrize("bits", [20, 24, 26])
@pytest.mark.parametrize("n, first", [(300, 0), (300, 170), (5000, 2)])
def test_attention_of_small_weights_beside_a_token_without_a_value(ops, dtype, fp8, bits, n, first):
    """A token that takes nearly all of the weight and whose value is zero: the output is made of weights of 2^-bits, which
    count as they are, not to the largest one's rounding (all logits but one are equal, so that errors would not cancel)."""
    pool = Pool([n, 40], 1, 128, 16, dtype, fp8, seed=34)
    g = torch.Generator(device="cuda").manual_seed(35)
    q = torch.randn(1, 1, 128, device="cuda", generator=g).expand(2, 4, 128).to(dtype)
    scale = 128 ** -0.5
    for r, at in ((0, first), (1, 3)):
        x = q[r, 0].double() * (bits * 0.6931471805599453 / (scale * q[r, 0].double().square().sum()))
        size = int(pool.lengths[r])
        pages, off = pool.table[r].long()[torch.arange(size, device="cuda") // 16], torch.arange(size, device="cuda") % 16
        sink = torch.zeros(size, 1, 1, device="cuda")
        sink[at] = 1
        for i, y in enumerate((sink * x.float(), torch.randn(size, 1, 128, device="cuda", generator=g).abs() * 1000 * (1 - sink))):
            if fp8:
                codes, s = quantised(y)
                pool.full[i].view(torch.uint8)[pages, :, off] = codes.view(torch.uint8)
                pool.scales[i][pages, :, off] = s
            else:
                pool.full[i][pages, :, off] = y.to(dtype)
    check(ops, pool, q, scale, attend(ops, pool, q, scale))


@pytest.mark.parametrize("fp8", [False, True])
def test_attention_of_values_near_the_largest(ops, fp8):
    """Values of 1.5e38 under logits that rise by up to 2^7.5 within a row: the output is 1.5e38 too, and no sum on the way
    there passes 3.4e38."""
    pool = Pool([200, 40], 1, 128, 16, BF, fp8, seed=36)
    g = torch.Generator(device="cuda").manual_seed(37)
    q = torch.randn(1, 1, 128, device="cuda", generator=g).expand(2, 4, 128).to(BF)
    x = q[0, 0].double() / (128 ** -0.5 * q[0, 0].double().square().sum()) * 0.6931471805599453  # a logit of 1, base 2
    for r, size in enumerate((200, 40)):
        pages, off = pool.table[r].long()[torch.arange(size, device="cuda") // 16], torch.arange(size, device="cuda") % 16
        z = torch.full((size, 1, 1), -40.0, device="cuda")
        for at, up in ((0, 0.0), (20, 5.0), (64, 7.0), (128, 7.5)):
            z[at:at + 1] = up
        values = torch.full((size, 1, 128), 1.5e38, device="cuda") * torch.where(torch.arange(128, device="cuda") % 3 > 0, 1, -1)
        for i, y in enumerate((z * x.float(), values)):
            if fp8:
                codes, s = quantised(y)
                pool.full[i].view(torch.uint8)[pages, :, off] = codes.view(torch.uint8)
                pool.scales[i][pages, :, off] = s
            else:
                pool.full[i][pages, :, off] = y.to(BF)
    check(ops, pool, q, 128 ** -0.5, attend(ops, pool, q, 128 ** -0.5))


def test_copies_beside_a_pool_that_holds_nothing(ops):
    """A pool of no layers, or of pages of no bytes, leaves the others' copies as they are."""
    p = torch.arange(2 * 6 * 8, dtype=torch.int32, device="cuda").view(2, 6, 8)
    want = p.clone()
    want[:, 4] = want[:, 1]
    ops.kv_copy_pages([p.new_empty(0, 6, 8), p, p.new_empty(3, 6, 0)], [1], [4])
    assert torch.equal(p, want)
    ops.kv_copy_pages([p.new_empty(0, 6, 8)], [1], [4])
    with pytest.raises(ValueError):
        ops.kv_copy_pages([p.new_empty(0, 6, 8), p], [1, 1], [4, 4])
    assert torch.equal(p, want)


# --- infinities and NaN that a row reads ---------------------------------------------------------------------------
INF, NAN = float("inf"), float("nan")


def without(pool, r, at):
    """The row's keys and values in 64 bits, position `at` left out, in check()'s place of the row."""
    class Rest(Pool):
        def __init__(self):
            self.scales = pool.scales

        def row(self, n):
            k, v = pool.row(r)
            keep = torch.arange(k.shape[1], device="cuda") != at
            return k[:, keep], v[:, keep]
    return Rest()


@pytest.mark.parametrize("dtype, fp8", [(BF, False), (FP16, False), (BF, True), (FP16, True)])
@pytest.mark.parametrize("n, at", [(100, 37), (5000, 4099)])
@pytest.mark.parametrize("what", [INF, -INF, NAN])
def test_attention_of_keys_with_infinities(ops, dtype, fp8, n, at, what):
    """A token of key head 1 whose key has an infinite (8-bit: a scale) or NaN part: logits of +inf and NaN make their
    heads NaN, one of -inf leaves the token out, and neither the other key head nor the other row see any of it."""
    pool = Pool([n, 100], 2, 128, 16, dtype, fp8, seed=41)
    q = torch.randn(2, 4, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(42)).to(dtype)
    q[0, 2], q[0, 3] = q[0, 2].abs() + 0.1, -q[0, 3].abs() - 0.1        # logits of both signs
    clean = attend(ops, pool, q, 0.09)
    page, off = pool.table[0, at // 16].long(), at % 16
    if fp8:
        pool.full[0].view(torch.uint8)[page, 1, off] = torch.full((128,), 0.5).to(E4M3).view(torch.uint8).cuda()
        pool.scales[0][page, 1, off] = what
    else:
        pool.full[0][page, 1, off, 5] = what
    got = attend(ops, pool, q, 0.09)
    assert torch.equal(got[0, :2], clean[0, :2]) and torch.equal(got[1], clean[1])
    lost = (2, 3) if what != what else (2,) if what > 0 else (3,)
    for h in (2, 3):
        if h in lost:
            assert got[0, h].isnan().all()
        else:  # check() of this head alone, over the row without the token
            check(ops, _one_head(without(pool, 0, at), 1), q[:1, h:h + 1], 0.09, got[:1, h:h + 1])


def _one_head(pool, head):
    row = pool.row
    pool.row = lambda n: tuple(x[head:head + 1] for x in row(n))
    return pool


@pytest.mark.parametrize("dtype, fp8", [(BF, False), (FP16, False), (BF, True), (FP16, True)])
@pytest.mark.parametrize("n, at", [(100, 37), (5000, 4099)])
@pytest.mark.parametrize("what", [INF, -INF, NAN])
def test_attention_of_values_with_infinities(ops, dtype, fp8, n, at, what):
    """A value's infinite or NaN part (8-bit: a NaN code, or the scale) reaches its dimension (the scale: every one) of the
    heads of its key head and nothing else."""
    pool = Pool([n, 100], 2, 128, 16, dtype, fp8, seed=43)
    q = torch.randn(2, 4, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(44)).to(dtype)
    clean = attend(ops, pool, q, 0.09)
    page, off = pool.table[0, at // 16].long(), at % 16
    dims = torch.zeros(128, dtype=torch.bool, device="cuda")
    if not fp8:
        pool.full[1][page, 1, off, 5] = what
        dims[5] = True
    elif what != what:
        pool.full[1].view(torch.uint8)[page, 1, off, 5] = 0x7F
        dims[5] = True
    else:
        pool.scales[1][page, 1, off] = what
        dims[:] = True
    got = attend(ops, pool, q, 0.09)
    assert torch.equal(got[0, :2], clean[0, :2]) and torch.equal(got[1], clean[1])
    assert not got[0, 2:][:, dims].isfinite().any()
    assert torch.equal(got[0, 2:][:, ~dims], clean[0, 2:][:, ~dims])


@pytest.mark.parametrize("dtype, fp8", [(BF, False), (FP16, False), (BF, True), (FP16, True)])
def test_attention_of_nothing_but_minus_infinity(ops, dtype, fp8):
    pool = Pool([1, 20], 1, 64, 16, dtype, fp8, seed=45)
    q = torch.ones(2, 2, 64, dtype=dtype, device="cuda")
    for r, size in ((0, 1), (1, 20)):
        for t in range(size):
            page = pool.table[r, t // 16].long()
            if fp8:
                pool.full[0].view(torch.uint8)[page, :, t % 16] = torch.ones(64).to(E4M3).view(torch.uint8).cuda()
                pool.scales[0][page, :, t % 16] = -INF
            else:
                pool.full[0][page, :, t % 16, 3] = -INF
    assert not attend(ops, pool, q, 0.125).any()
