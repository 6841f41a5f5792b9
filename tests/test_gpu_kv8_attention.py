"""Attention over the 8-bit cache through the C ABI against the formula in 64 bits."""

import numpy as np
import pytest
import torch

from fortai_amd import backend as B

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


class Case:
    """A filled cache, page tables and queries; what no token lies in holds NaN magnitudes."""

    def __init__(self, ctx, heads, kv, head, page, counts, lengths, dtype, gate=False, seed=0, spare=3, layers=1, loud=1.0):
        rng = np.random.default_rng(seed)
        self.ctx, self.heads, self.kv, self.head, self.page, self.dtype = ctx, heads, kv, head, page, dtype
        self.counts, self.lengths = list(counts), list(lengths)
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        need = [max(0, -(-(l + c) // page)) for l, c in zip(lengths, counts)]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages).astype(np.int32)
        self.tables = np.full((len(counts), max(max(need), 1) + 1), -1, dtype=np.int32)
        at = 0
        for s, n in enumerate(need):
            self.tables[s, :n] = order[at:at + n]
            at += n
        self.keys = rng.integers(-127, 128, (layers, self.pages, kv, page, head)).astype(np.int8)
        self.values = rng.integers(-127, 128, (layers, self.pages, kv, head, page)).astype(np.int8)
        self.key_max = rng.uniform(0.5, 3.0, (layers, self.pages, kv)).astype(np.float32)
        self.value_max = (rng.uniform(0.5, 3.0, (layers, self.pages, kv)) * loud).astype(np.float32)
        unused = order[at:]
        self.key_max[:, unused] = self.value_max[:, unused] = np.nan
        parts = 2 if gate else 1
        g = torch.Generator().manual_seed(seed)
        q = torch.randn(int(self.starts[-1]), heads, parts, head, generator=g)
        q[:, :, 0] *= torch.exp(torch.randn(1, heads, 1, generator=g))
        self.q, self.gate, self.scale = q.to(TYPES[dtype]), gate, head ** -0.5
        self.layers = layers

    def upload(self):
        storage = np.concatenate([a.reshape(-1).view(np.uint8) for a in (self.keys, self.values, self.key_max, self.value_max)])
        self.storage = torch.from_numpy(storage).cuda()
        self.cache = B.Kv8Cache(self.ctx, self.layers, self.pages, self.page, self.kv, self.head,
                                storage=self.storage.data_ptr(), storage_bytes=self.storage.numel())
        self.dev = [torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int32))).cuda() for a in (self.starts, self.lengths, self.tables)]
        self.batch = B.Kv8Batch(len(self.counts), int(self.starts[-1]), max(self.counts), *(d.data_ptr() for d in self.dev),
                                self.tables.shape[1])
        self.dq = self.q.cuda()
        self.out = torch.full((int(self.starts[-1]), self.heads, self.head), 77.0, dtype=TYPES[self.dtype], device="cuda")
        torch.cuda.synchronize()

    def run(self, layer=0, max_length=None):
        parts = 2 if self.gate else 1
        at = self.dq.data_ptr()
        self.cache.attention(layer, self.batch, at, self.heads, self.out.data_ptr(), self.scale,
                             max(l + c for l, c in zip(self.lengths, self.counts)) if max_length is None else max_length,
                             dtype=self.dtype, gate=at + self.head * self.dq.element_size() if self.gate else None,
                             query_head_pitch=parts * self.head, query_pitch=parts * self.heads * self.head)
        self.ctx.synchronize()
        return self.out.double().cpu().numpy()

    def formula(self, layer=0):
        """The result, and how far an fp32 computation of it may be off (see check)."""
        rows, group, page = int(self.starts[-1]), self.heads // self.kv, self.page
        want, bound = np.zeros((rows, self.heads, self.head)), np.zeros((rows, self.heads, self.head))
        q64 = self.q.double().numpy()
        for s, (count, length) in enumerate(zip(self.counts, self.lengths)):
            seen_pages = [(j, p) for j, p in enumerate(self.tables[s]) if 0 <= p < self.pages]
            for h in range(self.heads if seen_pages and length + count > 0 else 0):
                token = np.concatenate([np.arange(j * page, (j + 1) * page) for j, _ in seen_pages])
                pick = [p for _, p in seen_pages]
                k = (self.keys[layer, pick, h // group].astype(np.float64) * self.key_max[layer, pick, h // group].astype(np.float64)[:, None, None] / 127)
                v = (self.values[layer, pick, h // group].astype(np.float64) * self.value_max[layer, pick, h // group].astype(np.float64)[:, None, None] / 127)
                k, v = k.reshape(-1, self.head), v.transpose(0, 2, 1).reshape(-1, self.head)
                for i in range(count):
                    see = token <= length + i
                    if not see.any():
                        continue
                    q = q64[self.starts[s] + i, h, 0]
                    x = k[see] @ q * self.scale
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    row = self.starts[s] + i
                    want[row, h] = p @ v[see]
                    # scores: the queries keep 2^-23 of their row's largest; head fp32 additions; three roundings of the score
                    # (bf16 with more rows than 8 columns hold: two digits, 2^-16 of a power of two up to twice the largest)
                    size = abs(self.scale) * (np.abs(k[see]) @ np.abs(q))
                    kept = 2.0 ** -15 if self.dtype == "bf16" and self.single() else 2.0 ** -23
                    delta = np.max(abs(self.scale) * np.abs(q).max() * np.abs(k[see]).sum(1) * kept + size * self.head * 2.0 ** -24
                                   + (np.abs(x) + 150) * 3 * 2.0 ** -24)
                    # numerator and denominator: exp2 and the product with A, then sums of see terms in 16ths, joined
                    bound[row, h] = (p @ np.abs(v[see])) * (2 * delta + 8 * 2.0 ** -24 + 2 * (see.sum() / 16 + 64) * 2.0 ** -24)
                    # weights are pairs of fp16: the lower half's smallest step is 2^-24 of 2^-11, and the largest weight times
                    # magnitude stands at 2^11 at least (2^14 with few rows), so each is off by half of 2^-46 of that
                    bound[row, h] += see.sum() * 2.0 ** -47 * np.max(self.value_max[layer, pick, h // group])
        if self.gate:
            sigmoid = 1 / (1 + np.exp(-q64[:, :, 1]))
            want, bound = want * sigmoid, (bound + np.abs(want) * 2.0 ** -21) * sigmoid
        return want, bound

    def single(self):
        """Whether the kernel has weights as one fp16 number."""
        return self.dtype != "f32" and max(self.counts) * self.heads // self.kv > 8

    def check(self, got, layer=0):
        want, bound = self.formula(layer)
        if self.single():
            # more rows than 8 columns hold: p as one fp16 number, off by 2^-11 of itself, sum p = 1, |v| <= magnitude
            bound = bound + np.max(np.abs(self.value_max[np.isfinite(self.value_max)])) * 2.0 ** -11
        bound = bound + (np.abs(want) + bound) * HALF_STEP[self.dtype] + (2.0 ** -25 if self.dtype == "f16" else 1e-37)
        assert np.all(np.abs(got - want) <= bound), float(np.nanmax(np.abs(got - want) / bound))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,head,page", [(8, 2, 256, 64), (8, 2, 256, 16), (4, 4, 64, 32), (6, 2, 128, 64), (12, 1, 128, 16), (5, 5, 256, 32)])
def test_decode_steps(ctx, dtype, heads, kv, head, page):
    """One row a sequence: contexts of one token, at tile borders, empty batches' gaps, longer than one split."""
    c = Case(ctx, heads, kv, head, page, [1, 1, 0, 1, 1, 1], [0, 63, 9, 64, 200, 1500], dtype, gate=True, seed=heads + head)
    c.upload()
    c.check(c.run())
    c.cache.free()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,head,page,counts,lengths", [
    (8, 2, 256, 64, [5, 2, 3], [700, 0, 61]), (16, 4, 64, 16, [9, 1], [100, 3]), (4, 2, 128, 32, [17, 40, 1, 6], [0, 333, 5, 64]),
    (24, 3, 64, 64, [3, 3], [1000, 20]), (3, 3, 256, 64, [130], [70]), (8, 1, 128, 16, [33, 64], [511, 0])])
def test_several_rows(ctx, dtype, heads, kv, head, page, counts, lengths):
    """Drafts and prompt chunks: causal inside the rows, ragged, the last tiles of rows part empty."""
    c = Case(ctx, heads, kv, head, page, counts, lengths, dtype, gate=False, seed=len(counts) + head)
    c.upload()
    c.check(c.run())
    c.cache.free()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv,head,page,counts,lengths,gate", [
    (8, 2, 256, 64, [40, 2, 11], [700, 0, 61], True), (16, 4, 64, 16, [9, 1], [100, 3], False), (4, 2, 128, 32, [17, 40, 1, 6], [0, 333, 5, 64], True),
    (3, 3, 256, 16, [130], [70], False), (8, 1, 128, 16, [33, 64], [511, 0], True), (6, 2, 256, 32, [45, 0, 22], [-5, 9, 130], True),
    (32, 32, 64, 64, [70, 40, 66, 1], [0, 64, 30, 200], False), (32, 32, 256, 64, [70, 40, 66, 1], [0, 64, 30, 200], True)])
def test_many_rows(ctx, dtype, heads, kv, head, page, counts, lengths, gate):
    """As for long contexts, where 64 rows share a tile: max_length says so.  Split, and (32 heads) not split."""
    c = Case(ctx, heads, kv, head, page, counts, lengths, dtype, gate=gate, seed=heads + head + page)
    c.upload()
    c.check(c.run(max_length=1 << 20))
    c.cache.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("head", [64, 128, 256])
def test_many_rows_where_pages_are_odd(ctx, head, dtype):
    """Pages that are not there or hold zeros, unlike magnitudes, queries that are not finite, a negative scale."""
    c = Case(ctx, 8, 2, head, 16, [30, 19], [250, 90], dtype, seed=head)
    c.tables[0, 2:4] = [-1, c.pages + 5]
    c.key_max[:, c.tables[0, 5:8]] = 0.0
    c.value_max[:, c.tables[0, 6:9]] = 0.0
    c.value_max[:, c.tables[0, 10]] = 1e4
    c.value_max[:, c.tables[0, 11]] = 1e-30
    c.key_max[:, c.tables[1, 3]] *= 3.0
    c.scale = -c.scale
    c.q[45, 3, 0, 7] = float("inf")
    c.q[46, 0, 0, 0] = float("nan")
    c.upload()
    got = c.run(max_length=1 << 20)
    assert np.isnan(got[45, 3]).all() and np.isnan(got[46, 0]).all()
    c.q[45, 3] = c.q[46, 0] = 0.0
    want, _ = c.formula()
    got[45, 3], got[46, 0] = want[45, 3], want[46, 0]
    c.check(got)
    c.cache.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_max_length_only_cuts_the_work(ctx, dtype):
    c = Case(ctx, 8, 2, 128, 32, [2, 1, 3], [4000, 10, 700], dtype, gate=True, seed=4)
    c.upload()
    for most in (0, 1, 300, 4002, 10 ** 9):
        c.check(c.run(max_length=most))
    c.cache.free()


def test_long_context_split(ctx):
    c = Case(ctx, 4, 1, 256, 64, [2], [40000], "f32", seed=12)
    c.upload()
    c.check(c.run())
    c.cache.free()


@pytest.mark.parametrize("dtype,counts", [("f32", [1, 1, 1, 1]), ("bf16", [30, 25, 2, 1])])
def test_pages_that_are_not_there(ctx, dtype, counts):
    """Ids outside the pool, a table that ends early, tokens before the first, rows that see nothing: zeros there, and
    nothing else moves; rows of no sequence stay."""
    c = Case(ctx, 4, 2, 64, 16, counts, [100, 60, 5, 33], dtype, gate=True, seed=5)
    c.tables[0, 2] = -1
    c.tables[0, 4] = c.pages
    c.tables[1, :] = -7
    c.tables[3, 0] = 2 ** 31 - 1
    c.lengths[2] = -2 if dtype == "f32" else -1   # nothing to see (its first row, with two rows)
    c.upload()
    got = c.run()
    assert np.all(got[c.starts[1]:c.starts[2]] == 0) and np.all(got[c.starts[2]] == 0)
    c.check(got)
    # a batch whose arrays have rows behind the last sequence
    c.out.fill_(77.0)
    short = B.Kv8Batch(2, int(c.starts[-1]), max(counts), *(d.data_ptr() for d in c.dev), c.tables.shape[1])
    torch.cuda.synchronize()
    c.batch, all_rows = short, c.batch
    got = c.run()
    assert np.all(got[c.starts[2]:] == 77.0) and np.all(got[:c.starts[2]] != 77.0)
    # row starts that are out of range: no row is written twice or outside
    c.dev[0].copy_(torch.tensor([0, -5, 2 ** 31 - 1, 1, 0], dtype=torch.int32))
    c.out.fill_(77.0)
    torch.cuda.synchronize()
    c.batch = all_rows
    c.run()
    c.cache.free()


@pytest.mark.parametrize("dtype,count", [("f32", 1), ("bf16", 20)])
def test_pages_of_unlike_magnitudes(ctx, dtype, count):
    """Value pages from 1e-6 to 1e6, and of zeros only; key pages of zeros only."""
    c = Case(ctx, 2, 1, 64, 16, [count], [300], dtype, seed=6)
    c.value_max[0, :, 0] = 10.0 ** np.random.default_rng(1).uniform(-6, 6, c.pages)
    c.value_max[0, c.tables[0, 3]] = 0.0
    c.key_max[0, c.tables[0, 5]] = 0.0
    c.upload()
    c.check(c.run())
    c.value_max[:] = 0.0
    c.storage[c.storage.numel() - c.value_max.nbytes:] = 0
    torch.cuda.synchronize()
    assert np.all(c.run() == 0.0)
    # one loud page that the scores all but rule out, one quiet one that they choose
    c.value_max[0, :, 0] = 1e-4
    c.cache.free()


@pytest.mark.parametrize("dtype,counts", [("f32", [5, 1]), ("f16", [40, 3]), ("bf16", [1, 2]), ("bf16", [7, 1]), ("bf16", [70, 30])])
@pytest.mark.parametrize("head", [64, 256])
def test_pages_of_zeros_and_a_negative_scale(ctx, dtype, counts, head):
    """Magnitudes of zero: keys that score zero, values that add nothing but count; and the smallest scores win."""
    c = Case(ctx, 8, 2, head, 16, counts, [250, 90], dtype, seed=21, gate=True)
    c.scale = -c.scale
    c.key_max[:, c.tables[0, 1:4]] = 0.0
    c.value_max[:, c.tables[0, 3:9]] = 0.0
    c.value_max[:, c.tables[1, :2]] = 0.0
    c.upload()
    c.check(c.run())
    c.cache.free()


def test_a_quiet_page_that_is_chosen(ctx):
    """The page that takes the weight holds values 1e6 times smaller than the others."""
    c = Case(ctx, 1, 1, 64, 64, [1], [127], "f32", seed=3, spare=0)
    page = c.tables[0, 0]
    c.keys[0, c.tables[0, 1]] = 0
    c.q[0, 0, 0] = torch.from_numpy(c.keys[0, page, 0, 7].astype(np.float32)) / 20
    c.value_max[0, page, 0], c.value_max[0, c.tables[0, 1], 0] = 1e-3, 1e3
    c.upload()
    c.check(c.run())
    c.cache.free()


def test_queries_that_are_not_finite(ctx):
    c = Case(ctx, 4, 2, 64, 16, [4, 1], [50, 20], "f32", seed=7)
    c.upload()
    clean = c.run()
    c.dq[1, 2, 0, 5] = float("nan")
    c.dq[3, 0, 0, 1] = float("inf")
    torch.cuda.synchronize()
    got = c.run()
    bad = np.zeros(got.shape[:2], bool)
    bad[1, 2] = bad[3, 0] = True
    assert np.all(np.isnan(got[bad])) and np.array_equal(got[~bad], clean[~bad])
    c.cache.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("counts,max_length", [([9, 2], 40), ([45, 2], 40), ([45, 2], 1 << 20)])
def test_rows_without_tokens_are_zeros_whatever_they_ask(ctx, counts, max_length, dtype):
    """A sequence that begins before token 0: its first rows see nothing, NaN and infinities among their queries."""
    c = Case(ctx, 8, 2, 128, 16, counts, [-6, 20], dtype, seed=4)
    c.q[0], c.q[5, :, 0, 3] = float("nan"), float("-inf")
    c.upload()
    got = c.run(max_length=max_length)
    assert not got[:6].any()
    c.q[:6] = 0.0
    c.check(got)
    c.cache.free()


def test_pages_beyond_32_bits(ctx):
    """A pool of 5 GiB a layer: the second layer's last pages against the same tokens in its first ones."""
    layers, pages, page, kv, head, heads = 2, 40000, 64, 4, 256, 16
    cache = B.Kv8Cache(ctx, layers, pages, page, kv, head)
    g = torch.Generator().manual_seed(6)
    rows = 100
    k, v, q = (torch.randn(rows, n, head, generator=g).bfloat16().cuda() for n in (kv, kv, heads))
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, rows], [0], [[0, 1]], [[pages - 1, pages - 2]])]
    results = []
    for table in ints[2:]:
        batch = B.Kv8Batch(1, rows, rows, ints[0].data_ptr(), ints[1].data_ptr(), table.data_ptr(), 2)
        back = torch.zeros(2, rows, kv, head, dtype=torch.bfloat16, device="cuda")
        outs = torch.zeros(3, rows, heads, head, dtype=torch.bfloat16, device="cuda")
        torch.cuda.synchronize()
        cache.append(1, batch, k.data_ptr(), v.data_ptr(), dtype="bf16")
        cache.read(1, batch, back[0].data_ptr(), back[1].data_ptr(), dtype="bf16")
        for out, max_length in zip(outs, (100, 1 << 20)):
            cache.attention(1, batch, q.data_ptr(), heads, out.data_ptr(), 0.0625, max_length, dtype="bf16")
        last = B.Kv8Batch(1, rows, 2, ints[0].data_ptr(), ints[1].data_ptr(), table.data_ptr(), 2)
        cache.attention(1, last, q.data_ptr(), heads, outs[2].data_ptr(), 0.0625, 100, dtype="bf16")
        ctx.synchronize()
        results.append((back, outs))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    assert bool(results[0][1][:2].abs().amax(-1).all()) and bool(results[0][1][2, :2].abs().amax(-1).all())
    cache.copy_pages([pages - 1], [pages - 3])
    far = torch.tensor([[pages - 3, pages - 2]], dtype=torch.int32, device="cuda")
    batch = B.Kv8Batch(1, rows, rows, ints[0].data_ptr(), ints[1].data_ptr(), far.data_ptr(), 2)
    back = torch.zeros_like(results[0][0])
    torch.cuda.synchronize()
    cache.read(1, batch, back[0].data_ptr(), back[1].data_ptr(), dtype="bf16")
    ctx.synchronize()
    assert torch.equal(back, results[0][0])
    cache.free()


def test_pitches_and_layers(ctx):
    """Unaligned queries and outputs at pitches of their own; the second layer of two."""
    c = Case(ctx, 4, 2, 64, 16, [3, 2], [40, 100], "bf16", seed=8, layers=2)
    c.upload()
    c.check(c.run(layer=1), layer=1)
    rows = int(c.starts[-1])
    flat = torch.zeros(rows * 400 + 8, dtype=torch.bfloat16, device="cuda")
    q = torch.as_strided(flat, (rows, 4, 64), (397, 97, 1), 3)
    q.copy_(c.dq[:, :, 0])
    out = torch.full((rows, 300), 5.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    c.cache.attention(1, c.batch, q.data_ptr(), 4, out.data_ptr() + 2, c.scale, 102, dtype="bf16", query_pitch=397,
                      query_head_pitch=97, out_pitch=299)
    ctx.synchronize()
    got = torch.stack([out.reshape(-1)[1 + 299 * r:1 + 299 * r + 256] for r in range(rows)]).view(rows, 4, 64)
    assert torch.equal(got, c.out)
    untouched = torch.ones(rows * 300, dtype=torch.bool)
    for r in range(rows):
        untouched[1 + 299 * r:1 + 299 * r + 256] = False
    assert bool((out.reshape(-1).cpu()[untouched] == 5.0).all())
    c.cache.free()


def test_attention_refusals(ctx):
    c = Case(ctx, 4, 2, 64, 16, [2], [40], "f32", seed=9)
    c.upload()
    good = dict(layer=0, batch=c.batch, query=c.dq.data_ptr(), heads=4, out=c.out.data_ptr(), scale=0.1, max_length=42)
    c.cache.attention(**good)
    for bad in (dict(layer=1), dict(heads=5), dict(heads=0), dict(query=None), dict(out=None), dict(query=c.dq.data_ptr() + 2),
                dict(scale=float("nan")), dict(scale=float("inf")), dict(max_length=-1), dict(query_pitch=-1), dict(out_pitch=255),
                dict(gate=c.dq.data_ptr() + 1), dict(heads=65536), dict(batch=B.Kv8Batch(1, 2, 2, None, 16, 16, 1))):
        with pytest.raises(B.BackendError) as e:
            c.cache.attention(**{**good, **bad})
        assert e.value.code == B.INVALID
    c.cache.attention(**{**good, "batch": B.Kv8Batch(0, 0, 0, None, None, None, 0)})
    ctx.synchronize()
    c.cache.free()


def test_captured_calls_share_one_cache():
    """Append and two split attention calls in one graph, replayed with new lengths, queries and rows."""
    ctx = B.Context(0)
    c = Case(ctx, 8, 2, 128, 32, [1, 1], [3000, 1200], "f32", seed=10, spare=8)
    c.upload()
    other = torch.zeros_like(c.out)
    kv = torch.randn(2, 2, 2, 128, device="cuda")
    torch.cuda.synchronize()
    step = lambda out: c.cache.attention(0, c.batch, c.dq.data_ptr(), 8, out.data_ptr(), c.scale, 3001)
    append = lambda: c.cache.append(0, c.batch, kv.data_ptr(), kv.data_ptr() + 2 * 128 * 4, key_pitch=512, value_pitch=512)
    ctx.capture_begin()
    append()
    step(c.out)
    step(other)
    ctx.capture_end()
    for k in range(4):
        c.lengths = [3000 - 700 * k, 1200 - k]
        c.dev[1].copy_(torch.tensor(c.lengths, dtype=torch.int32))
        c.dq.copy_(torch.randn(c.dq.shape, generator=torch.Generator().manual_seed(k)))
        c.q = c.dq.cpu()
        kv.copy_(torch.randn(kv.shape, generator=torch.Generator().manual_seed(50 + k)))
        torch.cuda.synchronize()
        before = c.storage.clone()
        ctx.graph_launch()
        ctx.synchronize()
        got, again, after = c.out.clone(), other.clone(), c.storage.clone()
        c.storage.copy_(before)
        torch.cuda.synchronize()
        append()
        step(c.out)
        ctx.synchronize()
        assert torch.equal(got, c.out) and torch.equal(again, c.out) and torch.equal(after, c.storage)
        n = c.keys.size
        host = after.cpu().numpy()
        c.keys, c.values = host[:n].view(np.int8).reshape(c.keys.shape), host[n:2 * n].view(np.int8).reshape(c.values.shape)
        tops = host[2 * n:].view(np.float32).reshape(2, *c.key_max.shape)
        c.key_max, c.value_max = tops[0], tops[1]
        c.check(got.double().cpu().numpy())
    c.cache.free()
    ctx.close()
