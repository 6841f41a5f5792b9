"""The 8-bit paged cache through the C ABI: append, read and page copies against
their definition in 64 bits, code for code."""

import numpy as np
import pytest
import torch

from fortai_amd import backend as B

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


class Store:
    """The storage's planes on the host, and append by its definition."""

    def __init__(self, layers, pages, page, kv, head, seed):
        self.dims = (layers, pages, page, kv, head)
        rng = np.random.default_rng(seed)
        self.keys = rng.integers(-127, 128, (layers, pages, kv, page, head)).astype(np.int8)
        self.values = rng.integers(-127, 128, (layers, pages, kv, head, page)).astype(np.int8)
        self.key_max = rng.uniform(0.1, 3.0, (layers, pages, kv)).astype(np.float32)
        self.value_max = rng.uniform(0.1, 3.0, (layers, pages, kv)).astype(np.float32)

    def bytes(self):
        return np.concatenate([a.reshape(-1).view(np.uint8) for a in (self.keys, self.values, self.key_max, self.value_max)])

    def append(self, layer, k, v, starts, lengths, tables):
        """k, v [rows][kv][head] float64 (finite) of a ragged batch."""
        layers, pages, page, kv, head = self.dims
        for s in range(len(lengths)):
            n = starts[s + 1] - starts[s]
            for j in range(max(lengths[s], 0) // page, (lengths[s] + n + page - 1) // page):
                if j >= tables.shape[1] or not 0 <= tables[s, j] < pages:
                    continue
                first = j * page
                a, b = max(lengths[s], first, 0), min(lengths[s] + n, first + page)
                if a >= b:
                    continue
                old = a - first if lengths[s] > first else 0
                rows = slice(starts[s] + a - lengths[s], starts[s] + b - lengths[s])
                for x, codes, tops in ((k[rows], self.keys[layer, tables[s, j]], self.key_max),
                                       (v[rows], self.values[layer, tables[s, j]].transpose(0, 2, 1), self.value_max)):
                    for h in range(kv):
                        was = np.float64(tops[layer, tables[s, j], h]) if old else 0.0
                        top = max(was, np.abs(x[:, h]).max())
                        if old and top > was:
                            codes[h, :old] = np.rint(codes[h, :old].astype(np.float64) * was / top)
                        codes[h, a - first:b - first] = np.rint(x[:, h] * 127.0 / top) if top > 0 else 0
                        tops[layer, tables[s, j], h] = top


def to_device(*arrays):
    out = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays]
    torch.cuda.synchronize()
    return out


def batch_of(starts, lengths, tables, most=None):
    s, l, t = to_device(np.asarray(starts, np.int32), np.asarray(lengths, np.int32), np.asarray(tables, np.int32))
    rows = int(starts[-1])
    b = B.Kv8Batch(len(lengths), rows, rows if most is None else most, s.data_ptr(), l.data_ptr(), t.data_ptr(), t.shape[1])
    b.keep = (s, l, t)
    return b


def some_rows(rows, kv, head, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, 2, kv, head, generator=g) * torch.exp(torch.randn(rows, 2, kv, 1, generator=g))
    return x.to(TYPES[dtype])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,kv,head", [(16, 2, 64), (32, 3, 128), (64, 1, 256), (64, 4, 64), (16, 1, 256)])
def test_append_and_read(ctx, dtype, page, kv, head):
    """Lengths of zero, one, at and beside page borders; an empty sequence; a prompt over several pages."""
    counts = [1, 3, 0, 2 * page + 5, page, 7, 1]
    lengths = [0, page - 1, 5, 1, 0, page, 3 * page + 2]
    starts = np.concatenate([[0], np.cumsum(counts)])
    pages, pitch = 40, 6
    tables = np.random.default_rng(page + head).permutation(pages)[: len(counts) * 5].reshape(len(counts), 5).astype(np.int32)
    tables = np.pad(tables, ((0, 0), (0, 1)), constant_values=-1)
    store = Store(2, pages, page, kv, head, 5)
    storage, = to_device(store.bytes())
    assert B.Kv8Cache.bytes(2, pages, page, kv, head) == storage.numel()
    cache = B.Kv8Cache(ctx, 2, pages, page, kv, head, storage=storage.data_ptr(), storage_bytes=storage.numel())
    x = some_rows(starts[-1], kv, head, dtype, page * head)
    d = x.cuda()
    torch.cuda.synchronize()
    batch = batch_of(starts, lengths, tables)
    width, at = kv * head, d.data_ptr()
    cache.append(1, batch, at, at + width * d.element_size(), dtype=dtype, key_pitch=2 * width, value_pitch=2 * width)
    ctx.synchronize()
    x64 = x.double().numpy()
    store.append(1, x64[:, 0], x64[:, 1], starts, lengths, tables)
    assert np.array_equal(storage.cpu().numpy(), store.bytes())  # codes, magnitudes, and every byte beside them
    # all tokens read back, the old ones too
    ends = [l + c for l, c in zip(lengths, counts)]
    all_starts = np.concatenate([[0], np.cumsum(ends)])
    for out_dtype in ("f32", dtype):
        keys = torch.full((all_starts[-1], kv, head), 9.0, dtype=TYPES[out_dtype], device="cuda")
        values = torch.full((all_starts[-1], kv + 1, head), 9.0, dtype=TYPES[out_dtype], device="cuda")
        torch.cuda.synchronize()
        cache.read(1, batch_of(all_starts, [0] * len(ends), tables), keys.data_ptr(), values.data_ptr(), dtype=out_dtype,
                   value_pitch=(kv + 1) * head)
        ctx.synchronize()
        got_k, got_v = keys.double().cpu().numpy(), values.double().cpu().numpy()
        assert np.all(got_v[:, kv] == 9.0)
        for s, end in enumerate(ends):
            for t in range(end):
                p, slot, row = tables[s, t // page], t % page, all_starts[s] + t
                for got, code, top in ((got_k[row], store.keys[1, p, :, slot], store.key_max[1, p]),
                                       (got_v[row, :kv], store.values[1, p, :, :, slot], store.value_max[1, p])):
                    want = code.astype(np.float64) * top.astype(np.float64)[:, None] / 127.0
                    # two fp32 roundings (quotient, product), one to the type
                    assert np.all(np.abs(got - want) <= np.abs(want) * (2.01 * 2.0 ** -24 + 1.01 * HALF_STEP[out_dtype]) + 2.0 ** -25)
    cache.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_token_by_token(ctx, dtype):
    """Growing pages: the codes after each step are those of the definition."""
    page, kv, head, steps = 16, 2, 64, 40
    store = Store(1, 6, page, kv, head, 1)
    storage, = to_device(store.bytes())
    cache = B.Kv8Cache(ctx, 1, 6, page, kv, head, storage=storage.data_ptr(), storage_bytes=storage.numel())
    tables = np.array([[4, 0, 5], [2, 1, 3]], dtype=np.int32)
    x = some_rows(2 * steps, kv, head, dtype, 8)
    x[10] *= 50.0
    d, x64 = x.cuda(), x.double().numpy()
    torch.cuda.synchronize()
    for t in range(steps):
        at = d.data_ptr() + 2 * t * 2 * kv * head * d.element_size()
        cache.append(0, batch_of([0, 1, 2], [t, t + 3], tables, 1), at, at + kv * head * d.element_size(), dtype=dtype,
                     key_pitch=2 * kv * head, value_pitch=2 * kv * head)
        ctx.synchronize()
        store.append(0, x64[2 * t:2 * t + 2, 0], x64[2 * t:2 * t + 2, 1], [0, 1, 2], [t, t + 3], tables)
        assert np.array_equal(storage.cpu().numpy(), store.bytes()), t
    cache.free()


def test_append_ties_and_extreme_values(ctx):
    """Quotients that are halves exactly, magnitudes from subnormal to the largest, zeros, infinities and NaN."""
    page, kv, head = 16, 6, 64
    storage = torch.zeros(B.Kv8Cache.bytes(1, 1, page, kv, head), dtype=torch.uint8, device="cuda")
    cache = B.Kv8Cache(ctx, 1, 1, page, kv, head, storage=storage.data_ptr(), storage_bytes=storage.numel())
    x = torch.zeros(4, kv, head)
    ties = (torch.arange(head) - 32) + 0.5          # 127 x / A with A = 127: halves
    x[0, 0], x[1, 0, 0] = ties, 127.0
    x[0, 1], x[1, 1, 0] = ties * 3.0, 381.0          # halves of an A that is no power of two
    x[0, 2], x[1, 2, 0] = ties * 1e-42, 127e-42      # subnormal
    x[0, 3], x[1, 3, 0] = ties * 2.0 ** 120, 127.0 * 2.0 ** 120
    x[2, 4, :4] = torch.tensor([float("inf"), -float("inf"), float("nan"), 2.5])
    x[3, 4, 0] = -5.0
    x[2, 5, :3] = torch.tensor([float("inf"), float("nan"), -float("inf")])  # nothing finite but zeros
    d = x.cuda()
    torch.cuda.synchronize()
    cache.append(0, batch_of([0, 4], [0], [[0]]), d.data_ptr(), d.data_ptr())
    ctx.synchronize()
    host = storage.cpu().numpy()
    n = kv * page * head
    keys = host[:n].view(np.int8).reshape(kv, page, head)
    values = host[n:2 * n].view(np.int8).reshape(kv, head, page)
    tops = host[2 * n:].view(np.float32).reshape(2, kv)
    x64 = x.double().numpy()
    for h in range(4):
        top = np.abs(x64[:, h]).max()
        want = np.rint(x64[:, h] * 127.0 / top)
        assert np.array_equal(keys[h, :4], want) and np.array_equal(values[h, :, :4].T, want) and tops[0, h] == np.float32(top)
    assert keys[0, 0, 32] == 0 and keys[0, 0, 33] == 2  # 0.5 and 1.5: to even
    assert keys[4, 2, :4].tolist() == [127, -127, 0, round(127 * 2.5 / 5)] and keys[4, 3, 0] == -127 and tops[1, 4] == 5.0
    assert keys[5, 2, :3].tolist() == [127, 0, -127] and tops[0, 5] == 0.0
    cache.free()


def test_bad_rows_and_pages_reach_nothing_else(ctx):
    """Ids outside the pool, tokens before the first and past the table, row starts out of range: only what has a place is
    written, and read back as documented."""
    page, kv, head, pages = 16, 1, 64, 5
    store = Store(1, pages, page, kv, head, 3)
    guard = 4096
    whole = np.concatenate([np.full(guard, 0x5A, np.uint8), store.bytes(), np.full(guard, 0x5A, np.uint8)])
    storage, = to_device(whole)
    cache = B.Kv8Cache(ctx, 1, pages, page, kv, head, storage=storage.data_ptr() + guard, storage_bytes=len(whole) - 2 * guard)
    x = some_rows(60, kv, head, "f32", 4)
    d, x64 = x.cuda(), x.double().numpy()
    torch.cuda.synchronize()
    tables = np.array([[-1, 2, 99], [0, -7, 1], [3, 2 ** 31 - 1, 4]], dtype=np.int32)
    lengths, starts = [10, -5, 40], [0, 20, 40, 60]
    batch = batch_of(starts, lengths, tables)
    width = kv * head
    cache.append(0, batch, d.data_ptr(), d.data_ptr() + width * 4, key_pitch=2 * width, value_pitch=2 * width)
    ctx.synchronize()
    store.append(0, x64[:, 0], x64[:, 1], starts, lengths, tables)
    got = storage.cpu().numpy()
    assert np.array_equal(got[guard:-guard], store.bytes())
    assert np.all(got[:guard] == 0x5A) and np.all(got[-guard:] == 0x5A)
    keys, values = torch.full((60, kv, head), 3.0, device="cuda"), torch.full((60, kv, head), 3.0, device="cuda")
    torch.cuda.synchronize()
    cache.read(0, batch, keys.data_ptr(), values.data_ptr())
    ctx.synchronize()
    for s in range(3):
        for i in range(20):
            t, row = lengths[s] + i, keys[starts[s] + i].cpu().numpy()
            if t < 0:
                assert np.all(row == 3.0)
            elif t // page >= 3 or not 0 <= tables[s, t // page] < pages:
                assert np.all(row == 0.0)
            else:
                p = tables[s, t // page]
                assert np.allclose(row, store.keys[0, p, :, t % page] * (store.key_max[0, p] / 127.0)[:, None], rtol=1e-6)
    # rows past max_rows and past the batch are left out
    before = storage.clone()
    for bad_starts, most in (([5, 5, 3, 2 ** 31 - 1], 0), ([70, 80, 90, 60], 60)):
        b = batch_of(starts, [0, 0, 0], tables, most)
        b.keep[0].copy_(torch.tensor(bad_starts, dtype=torch.int32))
        torch.cuda.synchronize()
        cache.append(0, b, d.data_ptr(), d.data_ptr(), key_pitch=2 * width, value_pitch=2 * width)
        ctx.synchronize()
    assert torch.equal(storage, before)
    cache.free()


@pytest.mark.parametrize("page,kv,head,layers", [(16, 1, 64, 3), (64, 4, 256, 2), (32, 5, 128, 1)])
def test_copy_pages(ctx, page, kv, head, layers):
    pages = 1100
    if page == 64:
        pages = 40
    store = Store(layers, pages, page, kv, head, 6)
    storage, = to_device(store.bytes())
    cache = B.Kv8Cache(ctx, layers, pages, page, kv, head, storage=storage.data_ptr(), storage_bytes=storage.numel())
    order = np.random.default_rng(2).permutation(pages).astype(np.int32)
    half = pages // 2
    source, target = order[:half].copy(), order[half:2 * half].copy()
    source[1] = source[0]                              # the same page may be read twice
    cache.copy_pages(source, target)
    ctx.synchronize()
    for plane in (store.keys, store.values, store.key_max, store.value_max):
        plane[:, target] = plane[:, source]
    assert np.array_equal(storage.cpu().numpy(), store.bytes())
    cache.copy_pages([], [])
    for f, t in (([0], [0]), ([pages], [0]), ([0], [-1]), ([0, 1], [2, 2]), ([0, 1], [2, 0])):
        with pytest.raises(B.BackendError) as e:
            cache.copy_pages(f, t)
        assert e.value.code == B.INVALID
    ctx.synchronize()
    assert np.array_equal(storage.cpu().numpy(), store.bytes())
    cache.free()


def test_cache_refusals_and_own_storage(ctx):
    for bad in ((0, 4, 16, 1, 64), (1, 0, 16, 1, 64), (1, 4, 48, 1, 64), (1, 4, 16, 0, 64), (1, 4, 16, 1, 80), (4096, 2 ** 31 - 1, 64, 1024, 256)):
        with pytest.raises(B.BackendError) as e:
            B.Kv8Cache(ctx, *bad)
        assert e.value.code == B.INVALID
    storage = torch.zeros(B.Kv8Cache.bytes(1, 4, 16, 1, 64) + 16, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    for at, size in ((0, storage.numel() - 17), (8, storage.numel() - 8)):
        with pytest.raises(B.BackendError):
            B.Kv8Cache(ctx, 1, 4, 16, 1, 64, storage=storage.data_ptr() + at, storage_bytes=size)
    cache = B.Kv8Cache(ctx, 2, 4, 16, 1, 64)
    rows = torch.randn(4, 64, device="cuda")
    out = torch.empty(2, 4, 64, device="cuda")
    batch = batch_of([0, 4], [0], [[3]])
    torch.cuda.synchronize()
    for layer, b, k, more in ((2, batch, rows.data_ptr(), {}), (-1, batch, rows.data_ptr(), {}), (0, batch, None, {}),
                              (0, batch, rows.data_ptr() + 1, {}), (0, batch, rows.data_ptr(), dict(key_pitch=-1)),
                              (0, B.Kv8Batch(1, 4, 5, 16, 16, 16, 1), rows.data_ptr(), {}),
                              (0, B.Kv8Batch(1, 4, 4, None, 16, 16, 1), rows.data_ptr(), {}),
                              (0, B.Kv8Batch(1, 4, 4, 16, 16, 16, 0), rows.data_ptr(), {})):
        with pytest.raises(B.BackendError) as e:
            cache.append(layer, b, k, rows.data_ptr(), **more)
        assert e.value.code == B.INVALID
        with pytest.raises(B.BackendError):
            cache.read(layer, b, k, out.data_ptr(), **more)
    with pytest.raises(B.BackendError):
        cache.read(0, batch, out.data_ptr(), out.data_ptr(), key_pitch=63)
    cache.append(0, B.Kv8Batch(0, 0, 0, None, None, None, 0), None, None)  # nothing to do
    cache.append(1, batch, rows.data_ptr(), rows.data_ptr())
    for layer in (0, 1):
        cache.read(layer, batch, out[0].data_ptr(), out[1].data_ptr())
        ctx.synchronize()
        if layer == 0:
            assert bool((out == 0).all())  # cleared storage, the other layer untouched
        else:
            assert float((out - rows).abs().max()) <= float(rows.abs().max()) / 254 * 1.0001
    cache.free()
