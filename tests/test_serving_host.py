"""Host logic of the serving operators, without a GPU: page bookkeeping, argument
checks, the frequencies of rotary positions, and how ragged batches with bad
numbers are brought into range."""

import ctypes as C
import math
import os
import random
import subprocess

import numpy as np
import pytest

from fortai_amd import backend as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "fortai_amd", "csrc")


def compiled(tmp_path, source):
    path, so = tmp_path / "host.cpp", str(tmp_path / "libhost.so")
    path.write_text(source)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, str(path), "-o", so], check=True)
    return C.CDLL(so)


# ------------------------------------------------------------- pages
class Model:
    """Page bookkeeping as sets of tokens: what every sequence's slots must hold."""

    def __init__(self, pages, page, sequences, pitch):
        self.page, self.pitch = page, pitch
        self.content = {p: {} for p in range(pages)}  # page -> slot -> token
        self.tokens = [[] for _ in range(sequences)]


def write(model, pool, seq, count, stamp):
    """extend, copy, write the new tokens through the table; the tokens are unique stamps."""
    pairs = pool.extend(seq, count)
    for f, t in pairs:
        model.content[t] = dict(model.content[f])
    table = pool.tables([seq])[0]
    for k in range(count):
        at = len(model.tokens[seq])
        model.tokens[seq].append((stamp, k))
        model.content[table[at // model.page]][at % model.page] = (stamp, k)


def consistent(model, pool):
    held = set()
    for seq, tokens in enumerate(model.tokens):
        assert pool.length(seq) == len(tokens)
        table = pool.tables([seq])[0]
        need = -(-len(tokens) // model.page)
        assert all(t >= 0 for t in table[:need]) and all(t == -1 for t in table[need:])
        assert len(set(table[:need])) == need
        held |= set(table[:need].tolist())
        for at, token in enumerate(tokens):
            assert model.content[table[at // model.page]][at % model.page] == token
    assert pool.free_count() == len(model.content) - len(held)


@pytest.mark.parametrize("seed", range(6))
def test_pages_against_a_model(seed):
    """Random extends, forks, truncations and compactions: every sequence keeps its own tokens."""
    rng = random.Random(seed)
    pages, page, sequences, pitch = rng.choice([(40, 16, 6, 12), (9, 32, 3, 5), (200, 64, 10, 20)])
    pool, model = B.Kv8Pages(pages, page, sequences, pitch), Model(pages, page, sequences, pitch)
    for step in range(300):
        seq, what = rng.randrange(sequences), rng.random()
        if what < 0.5:
            count = rng.choice([0, 1, 1, 2, 5, page, 3 * page + 1])
            before = [t.copy() for t in pool.tables(range(sequences))], pool.free_count()
            try:
                write(model, pool, seq, count, step)
            except B.BackendError as e:
                assert e.code == B.INVALID
                after = pool.tables(range(sequences)), pool.free_count()
                assert before[1] == after[1] and all((a == b).all() for a, b in zip(before[0], after[0]))
        elif what < 0.65:
            other = rng.randrange(sequences)
            length = rng.randint(0, len(model.tokens[seq]))
            if other == seq or model.tokens[other]:
                with pytest.raises(B.BackendError):
                    pool.fork(seq, other, length)
            else:
                pool.fork(seq, other, length)
                model.tokens[other] = model.tokens[seq][:length]
        elif what < 0.9:
            length = rng.randint(0, len(model.tokens[seq]))
            pool.truncate(seq, length)
            del model.tokens[seq][length:]
        else:
            f, t = pool.compact(rng.choice([None, 1, 3]))
            assert len(set(t.tolist())) == len(t) and not set(f.tolist()) & set(t.tolist()) and all(f > t)
            for a, b in zip(f.tolist(), t.tolist()):
                model.content[b] = dict(model.content[a])
                model.content[a] = {}
        consistent(model, pool)
    f, t = pool.compact()
    for a, b in zip(f.tolist(), t.tolist()):
        model.content[b] = dict(model.content[a])
    live = pages - pool.free_count()
    table = pool.tables(range(sequences))
    assert table.max(initial=-1) < live and len(pool.compact()[0]) == 0
    consistent(model, pool)
    for seq in range(sequences):
        pool.truncate(seq)
    assert pool.free_count() == pages
    pool.free()


def test_pages_share_until_written():
    pool = B.Kv8Pages(8, 16, 3, 4)
    assert pool.extend(0, 20) == [] and pool.free_count() == 6
    pool.fork(0, 1, 20)
    pool.fork(0, 2, 16)
    assert pool.free_count() == 6
    assert pool.extend(2, 1) == []                 # at a page's end: a page of its own, nothing to copy
    assert pool.extend(1, 1) == [(1, 3)]           # inside the shared page: its own copy
    assert pool.extend(0, 1) == []                 # now alone on it
    assert pool.tables([0, 1, 2])[:, :3].tolist() == [[0, 1, -1], [0, 3, -1], [0, 2, -1]]
    pool.truncate(1, 3)                            # back into the page that all three share
    assert pool.extend(1, 1) == [(0, 3)]
    pool.free()


def test_pages_refusals():
    for bad in ((0, 16, 1, 1), (1, 17, 1, 1), (1, 16, 0, 1), (1, 16, 1, 0), (1, 16, 1, (1 << 24) + 1)):
        with pytest.raises(B.BackendError):
            B.Kv8Pages(*bad)
    pool = B.Kv8Pages(4, 16, 2, 3)
    for call in (lambda: pool.extend(2, 1), lambda: pool.extend(-1, 1), lambda: pool.extend(0, -1),
                 lambda: pool.extend(0, 49), lambda: pool.fork(0, 0, 0), lambda: pool.fork(0, 1, 1),
                 lambda: pool.truncate(0, 1), lambda: pool.truncate(0, -1), lambda: pool.tables([2])):
        with pytest.raises(B.BackendError) as e:
            call()
        assert e.value.code == B.INVALID
    assert pool.length(2) == -1 and pool.length(0) == 0 and pool.free_count() == 4
    pool.extend(0, 48)
    with pytest.raises(B.BackendError):
        pool.extend(1, 17)                         # one page left
    assert pool.length(1) == 0 and pool.free_count() == 1
    lib = B.load()
    assert lib.fortai_hip_kv8_pages_destroy(None) == 0 and lib.fortai_hip_kv8_pages_length(None, 0) == -1
    pool.free()


def test_the_stub_counts_no_pages(tmp_path):
    """Without the library: a length and a count of -1, as the library answers where there is no pool."""
    so = str(tmp_path / "libstub.so")
    subprocess.run(["gcc", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "include"),
                    os.path.join(ROOT, "fortai_amd", "fortran", "fortai_hip_stub.c"), "-o", so], check=True)
    for lib in (C.CDLL(so), B.load()):
        lib.fortai_hip_kv8_pages_length.restype = C.c_int64
        lib.fortai_hip_kv8_bytes.restype = C.c_size_t
        assert lib.fortai_hip_kv8_pages_length(None, 0) == -1 and lib.fortai_hip_kv8_pages_free_count(None) == -1
        assert lib.fortai_hip_kv8_bytes(1, 0, 16, 1, 64) == 0


# ------------------------------------------------------------- checks
def test_rope_checks_and_frequencies(tmp_path):
    lib = compiled(tmp_path, '''
#include "serving_checks.h"
using namespace fortai_hip;
extern "C" {
const char *create(int d, double base, int scaling, double factor, int original, double fast, double slow, double att) {
    return check_rope_create(d, base, scaling, factor, original, fast, slow, att); }
void turns(int d, double base, int scaling, double factor, int original, double fast, double slow, double *out) {
    rope_turns(d, base, scaling, factor, original, fast, slow, out); }
int touch(int64_t rows, int64_t heads, int64_t head, int64_t rp, int64_t hp) { return apart(rows, heads, head, rp, hp); }
}''')
    lib.create.restype = C.c_char_p
    lib.create.argtypes = [C.c_int, C.c_double, C.c_int, C.c_double, C.c_int, C.c_double, C.c_double, C.c_double]
    assert lib.create(64, 1e4, 0, 0.0, 0, 0.0, 0.0, 1.0) is None
    assert lib.create(64, 1e4, 2, 4.0, 4096, 32.0, 1.0, 1.1) is None
    for bad in ((63, 1e4, 0, 1, 0, 0, 0, 1), (64, -1, 0, 1, 0, 0, 0, 1), (64, 1e4, 3, 1, 0, 0, 0, 1), (64, 1e4, 1, 0, 0, 0, 0, 1),
                (64, 1e4, 2, 4, 0, 32, 1, 1), (64, 1e4, 2, 4, 4096, 1, 1, 1), (64, 1.0, 2, 4, 4096, 32, 1, 1),
                (64, float("inf"), 0, 1, 0, 0, 0, 1), (64, 1e4, 0, 1, 0, 0, 0, 0)):
        assert lib.create(*bad), bad
    out = (C.c_double * 32)()
    lib.turns.argtypes = [C.c_int, C.c_double, C.c_int, C.c_double, C.c_int, C.c_double, C.c_double, C.c_void_p]
    lib.turns(64, 1e4, 0, 1.0, 0, 32.0, 1.0, out)
    want = np.array([1e4 ** (-2 * i / 64) / (2 * math.pi) for i in range(32)])
    assert np.allclose(out[:], want, rtol=1e-14)
    lib.turns(64, 1e4, 2, 8.0, 4096, 32.0, 1.0, out)
    ratio = np.array(out[:]) / want
    assert np.allclose(ratio[:5], 1.0) and np.allclose(ratio[-5:], 1 / 8) and np.all(np.diff(ratio) <= 1e-12)
    lib.touch.argtypes = [C.c_int64] * 5
    assert lib.touch(3, 4, 64, 256, 64) and lib.touch(3, 4, 64, 64, 192) and lib.touch(1, 4, 64, 0, 64) and lib.touch(3, 1, 64, 64, 0)
    assert not lib.touch(3, 4, 64, 255, 64) and not lib.touch(3, 4, 64, 64, 191) and not lib.touch(3, 4, 64, 256, 63)
    assert not lib.touch(2, 1, 64, 0, 0)


def test_cache_checks(tmp_path):
    lib = compiled(tmp_path, '''
#include "serving_checks.h"
using namespace fortai_hip;
static Kv8Shape shape(int layers, int pages, int page, int heads, int head) {
    Kv8Shape s; s.layers = layers; s.pages = pages; s.page_tokens = page; s.kv_heads = heads; s.head = head; return s; }
extern "C" {
size_t bytes(int l, int p, int t, int h, int d) { return kv8_bytes(shape(l, p, t, h, d)); }
const char *batch(int n, int rows, int most, int pitch, const void *a, const void *b, const void *c) {
    return check_kv8_batch(n, rows, most, pitch, a, b, c); }
const char *rows(int layer, int dtype, const void *k, int64_t kp, const void *v, int64_t vp, int written) {
    return check_kv8_rows(shape(2, 8, 16, 2, 64), layer, dtype, k, kp, v, vp, written != 0); }
const char *pairs(const int32_t *f, const int32_t *t, int n, int pages) { return check_page_pairs(f, t, n, pages); }
}''')
    lib.bytes.restype = C.c_size_t
    for f in (lib.batch, lib.rows, lib.pairs):
        f.restype = C.c_char_p
    assert lib.bytes(3, 5, 16, 2, 64) == 3 * 5 * 2 * (2 * 16 * 64 + 8)
    assert lib.bytes(4096, 2 ** 31 - 1, 64, 1024, 256) == 0  # past any memory: refused, not wrapped
    for bad in ((0, 5, 16, 2, 64), (1, 0, 16, 2, 64), (1, 5, 24, 2, 64), (1, 5, 16, 0, 64), (1, 5, 16, 2, 96), (1, 5, 16, 1025, 64)):
        assert lib.bytes(*bad) == 0
    lib.batch.argtypes = [C.c_int] * 4 + [C.c_void_p] * 3
    assert lib.batch(2, 5, 3, 4, 16, 16, 16) is None and lib.batch(0, 0, 0, 0, None, None, None) is None
    for bad in ((-1, 5, 3, 4, 16, 16, 16), (2, -1, 0, 4, 16, 16, 16), (2, 5, 6, 4, 16, 16, 16), (2, 5, 3, 0, 16, 16, 16),
                (2, 5, 3, 4, None, 16, 16), (2, 5, 3, 4, 16, 18, 16), (16385, 5, 3, 4, 16, 16, 16), (2, 1 << 24, 3, 4, 16, 16, 16)):
        assert lib.batch(*bad), bad
    lib.rows.argtypes = [C.c_int, C.c_int, C.c_void_p, C.c_int64, C.c_void_p, C.c_int64, C.c_int]
    assert lib.rows(1, 2, 16, 0, 16, 128, 0) is None and lib.rows(1, 2, 18, 128, 16, 500, 1) is None
    for bad in ((2, 0, 16, 128, 16, 128, 0), (-1, 0, 16, 128, 16, 128, 0), (0, 3, 16, 128, 16, 128, 0), (0, 0, None, 128, 16, 128, 0),
                (0, 0, 18, 128, 16, 128, 0), (0, 0, 16, -1, 16, 128, 0), (0, 0, 16, 127, 16, 128, 1), (0, 0, 16, 1 << 32, 16, 128, 0)):
        assert lib.rows(*bad), bad
    pairs = lambda f, t: lib.pairs((C.c_int32 * len(f))(*f), (C.c_int32 * len(t))(*t), len(f), 8)
    assert pairs([7], [0]) is None and pairs([5, 5, 6], [0, 1, 2]) is None
    for f, t in (([8], [0]), ([0], [-1]), ([3], [3]), ([1, 2], [0, 0]), ([1, 2], [0, 1]), ([0, 1, 2], [3, 4, 0])):
        assert pairs(f, t), (f, t)


def test_batches_with_bad_numbers_stay_in_range(tmp_path):
    """Row starts out of order or out of range, lengths at the ends of 32 bits, ids outside the pool."""
    lib = compiled(tmp_path, '''
#include "kv8_device.h"
using namespace fortai_hip;
extern "C" void look(const int32_t *starts, const int32_t *lengths, const int32_t *tables, int n, int rows, int most, int pitch,
    int seq, int index, int pages, int *out) {
    Kv8Rows r; r.starts = starts; r.lengths = lengths; r.tables = tables; r.sequences = n; r.rows = rows; r.max_rows = most; r.pitch = pitch;
    r.range(seq, out, out + 1); out[2] = r.length(seq); out[3] = r.page(seq, index, pages); }''')
    starts = np.array([0, 4, 2, 2 ** 31 - 1, -5, 10], dtype=np.int32)
    lengths = np.array([0, -1, 2 ** 31 - 1, -2 ** 31, 7], dtype=np.int32)
    tables = np.array([[0, 1], [5, -1], [2 ** 31 - 1, -2 ** 31], [3, 4], [4, 0]], dtype=np.int32)
    out = np.zeros(4, dtype=np.int32)
    ptr = lambda a: C.c_void_p(a.ctypes.data)
    for seq in range(5):
        for index in (-1, 0, 1, 2, 2 ** 30, -2 ** 31):
            lib.look(ptr(starts), ptr(lengths), ptr(tables), 5, 10, 4, 2, seq, index, 5, ptr(out))
            begin, count, length, page = out.tolist()
            assert 0 <= begin <= 10 and 0 <= count <= 4 and begin + count <= 10
            assert -2 ** 30 <= length <= 2 ** 30
            want = tables[seq, index] if 0 <= index < 2 and 0 <= tables[seq, index] < 5 else -1
            assert page == want
    lib.look(ptr(starts), ptr(lengths), ptr(tables), 5, 10, 4, 2, 0, 0, 5, ptr(out))
    assert out[:2].tolist() == [0, 4]
    lib.look(ptr(starts), ptr(lengths), ptr(tables), 5, 10, 4, 2, 1, 0, 5, ptr(out))
    assert out[1] == 0  # starts that fall: no rows
    lib.look(ptr(starts), ptr(lengths), ptr(tables), 5, 10, 4, 2, 4, 0, 5, ptr(out))
    assert out[:2].tolist() == [0, 4]  # from below zero: clipped to the batch, then to max_rows


def test_attention_checks_and_plan(tmp_path):
    lib = compiled(tmp_path, '''
#include "kv8_device.h"
#include "serving_checks.h"
using namespace fortai_hip;
extern "C" {
const char *check(int kv, int layer, int dtype, int rows, int most, const void *q, int64_t qp, int64_t qh, const void *gate, int heads,
    float scale, int length, const void *out, int64_t op) {
    Kv8Shape s; s.layers = 2; s.pages = 8; s.page_tokens = 16; s.kv_heads = kv; s.head = 64;
    return check_kv8_attention(s, layer, dtype, rows, most, q, qp, qh, gate, heads, scale, length, out, op); }
void plan(int fp32, int head, int sequences, int kv, int64_t rows, int64_t length, int *out) {
    const Kv8Plan p = kv8_plan(fp32 != 0, head, sequences, kv, rows, length);
    out[0] = p.rows; out[1] = p.row_tiles; out[2] = p.splits; out[3] = kKv8PartialRows; out[4] = kKv8MaxSplits; }
}''')
    lib.check.restype = C.c_char_p
    lib.check.argtypes = [C.c_int] * 5 + [C.c_void_p, C.c_int64, C.c_int64, C.c_void_p, C.c_int, C.c_float, C.c_int, C.c_void_p, C.c_int64]
    good = dict(kv=2, layer=1, dtype=2, rows=9, most=5, q=16, qp=512, qh=64, gate=None, heads=8, scale=0.125, length=100, out=16, op=512)
    check = lambda **kw: lib.check(*{**good, **kw}.values())
    assert check() is None and check(qp=0, qh=0, gate=18, length=0, scale=-1.0) is None and check(rows=1, most=1, op=0) is None
    assert check(kv=1024, heads=1024, rows=8 * 63, most=8 * 63, op=1 << 16) is None  # 63 tiles of 1024 heads are within the grid
    nan = float("nan")
    for bad in (dict(layer=2), dict(layer=-1), dict(dtype=3), dict(heads=9), dict(heads=0), dict(heads=65536), dict(scale=nan),
                dict(scale=float("inf")), dict(length=-1), dict(q=None), dict(out=None), dict(q=17), dict(gate=17), dict(out=17),
                dict(qp=-1), dict(qh=1 << 32), dict(op=511), dict(op=1 << 32), dict(kv=1024, heads=1024, rows=8 * 64, most=8 * 64, op=1 << 16),
                dict(rows=1 << 22, most=1 << 22, heads=64)):
        assert check(**bad), bad
    out = (C.c_int * 5)()
    lib.plan.argtypes = [C.c_int] * 4 + [C.c_int64] * 2 + [C.c_void_p]
    rng = random.Random(1)
    for _ in range(3000):
        fp32, head, kv = rng.randrange(2), rng.choice([64, 128, 256]), rng.choice([1, 2, 3, 8, 64, 1024])
        sequences, rows, length = rng.choice([1, 2, 37, 16384]), int(2 ** rng.uniform(0, 23)), int(2 ** rng.uniform(0, 31)) - 1
        lib.plan(fp32, head, sequences, kv, rows, length, out)
        tile, tiles, splits, room, most = out[:]
        few = 8 if fp32 or rows <= 8 else 16
        assert tile in ((few,) if rows <= 2 * few else (few, 4 * few)) and tiles == -(-rows // tile)
        assert 1 <= splits <= most and (splits == 1 or splits * tiles * tile * kv * sequences <= room)
        assert splits <= max(1, -(-length // (128 if tile > 16 else 256)))  # every split has work for its waves


def test_verify_checks(tmp_path):
    lib = compiled(tmp_path, '''
#include "serving_checks.h"
using namespace fortai_hip;
extern "C" {
const char *create(int rows, int sequences, int vocab) { return check_verifier(rows, sequences, vocab); }
int chunk(int rows, int vocab) { return verify_chunk(rows, vocab); }
const char *check(int dtype, const void *t, int64_t tp, const void *d, int64_t dp, const void *tokens, const void *u, const void *temp,
    int sequences, const void *starts, int rows, const void *e, const void *a, const void *l) {
    return check_verify(40, 8, 1000, dtype, t, tp, d, dp, tokens, u, temp, sequences, starts, rows, e, a, l); }
}''')
    lib.create.restype = lib.check.restype = C.c_char_p
    assert lib.create(1, 1, 1) is None and lib.create(65535, 65535, 1 << 28) is None
    for bad in ((0, 1, 1), (65536, 1, 1), (1, 0, 1), (1, 65536, 1), (1, 1, 0), (1, 1, (1 << 28) + 1)):
        assert lib.create(*bad), bad
    assert lib.chunk(1, 1) == 1024 and lib.chunk(40, 248320) == 4096 and lib.chunk(65535, 1 << 28) == 4096
    lib.check.argtypes = [C.c_int, C.c_void_p, C.c_int64, C.c_void_p, C.c_int64, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_void_p,
                          C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]
    good = dict(dtype=0, target=16, tp=1000, draft=None, dp=0, tokens=16, u=16, temp=None, sequences=8, starts=16, rows=40, e=16, a=16,
                l=None)
    check = lambda **kw: lib.check(*{**good, **kw}.values())
    assert check() is None and check(draft=16, dp=1000, temp=16, l=16) is None and check(rows=0, target=None, tokens=None, u=None, e=None) is None
    assert check(sequences=0, starts=None) is None and check(dtype=1, target=18) is None
    for bad in (dict(dtype=3), dict(sequences=9), dict(sequences=-1), dict(rows=41), dict(rows=-1), dict(starts=None), dict(a=None),
                dict(target=None), dict(tokens=None), dict(u=None), dict(e=None), dict(target=18), dict(draft=17, dp=1000), dict(tokens=20),
                dict(u=18), dict(temp=18), dict(starts=18), dict(e=20), dict(a=18), dict(l=18), dict(tp=999), dict(tp=1 << 32),
                dict(draft=16, dp=999), dict(draft=16, dp=1 << 32)):
        assert check(**bad), bad


def test_fortran_pages_and_refusals():
    """The Fortran module's page bookkeeping and its refusals, through the library as built."""
    from fortai_amd import build
    r = subprocess.run([build.SERVING_SMOKE], capture_output=True, text=True, timeout=120)
    print(r.stdout, r.stderr)
    assert r.returncode == 0 and "fortran serving smoke ok" in r.stdout
