"""Host logic of the operators around a step's products, without a GPU: argument checks, the bytes of a delta rule's
cache, which sequences share pages, and how attention over shared pages is cut."""

import ctypes as C
import itertools
import random

import numpy as np
import pytest

from fortai_amd import backend as B
from test_serving_host import compiled

NAN = float("nan")


def arrays(struct, pointers, pitches):
    """A ctypes twin of a struct of pointers, then pitches."""
    return type(struct, (C.Structure,), {"_fields_": [(n, C.c_void_p) for n in pointers] + [(n, C.c_int64) for n in pitches]})


def test_norm_tokens_checks(tmp_path):
    lib = compiled(tmp_path, '''
#include "step_checks.h"
using namespace fortai_hip;
extern "C" {
const char *norm(int dtype, int rows, int width, int group, float eps, const NormTokensArrays *a) {
    return check_norm_tokens(dtype, rows, width, group, eps, *a); }
const char *read(int dtype, int rows, int width, const void *tokens, const void *out, int64_t pitch) {
    return check_tokens_read(dtype, rows, width, tokens, out, pitch); }
}''')
    lib.norm.restype = lib.read.restype = C.c_char_p
    A = arrays("A", ["x", "residual", "sum", "norm", "gate", "output", "tokens"], ["xp", "rp", "sp", "gp", "op"])
    lib.norm.argtypes = [C.c_int] * 4 + [C.c_float, C.POINTER(A)]
    good = dict(dtype=1, rows=4, width=320, group=64, eps=1e-6)
    data = dict(x=16, residual=18, sum=18, norm=20, gate=22, output=24, tokens=32, xp=0, rp=640, sp=640, gp=0, op=320)

    def check(**kw):
        return lib.norm(*{k: kw.get(k, v) for k, v in good.items()}.values(), A(**{k: kw.get(k, v) for k, v in data.items()}))
    assert check() is None
    assert check(group=320, residual=None, sum=None, gate=None, output=None) is None and check(tokens=None) is None
    assert check(norm=None, eps=0.0) is None and check(rows=0, x=None) is None and check(rows=1, sp=0, op=0) is None
    assert check(rows=1 << 23, width=1 << 20, group=256, rp=1 << 20, sp=1 << 20, op=1 << 20) is None
    for bad in (dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(rows=(1 << 23) + 1), dict(width=0), dict(width=31), dict(width=48),
                dict(width=(1 << 20) + 32, group=32), dict(group=0), dict(group=16), dict(group=128), dict(group=-32), dict(eps=0.0),
                dict(eps=NAN), dict(x=None), dict(output=None, tokens=None), dict(x=17), dict(residual=17), dict(sum=19), dict(norm=18),
                dict(gate=17), dict(output=17), dict(tokens=24), dict(xp=-1), dict(xp=1 << 32), dict(rp=-1), dict(gp=1 << 32),
                dict(sp=319), dict(op=319), dict(op=1 << 32), dict(rp=960), dict(x=18, residual=16, xp=320)):
        assert check(**bad), bad
    ok = dict(dtype=2, rows=3, width=64, tokens=16, out=18, pitch=64)
    read = lambda **kw: lib.read(*{**ok, **kw}.values())
    lib.read.argtypes = [C.c_int] * 3 + [C.c_void_p] * 2 + [C.c_int64]
    assert read() is None and read(rows=1, pitch=0) is None and read(rows=0, tokens=None) is None
    for bad in (dict(dtype=3), dict(rows=-1), dict(rows=(1 << 23) + 1), dict(width=33), dict(width=0), dict(tokens=None), dict(out=None),
                dict(tokens=24), dict(out=17), dict(pitch=63), dict(pitch=-1), dict(pitch=1 << 32)):
        assert read(**bad), bad


def test_logit_rules_checks(tmp_path):
    lib = compiled(tmp_path, '''
#include "step_checks.h"
using namespace fortai_hip;
extern "C" const char *rules(int dtype, int rows, int vocab, int sequences, int window, int masks, const LogitRulesArrays *a) {
    return check_logit_rules(dtype, rows, vocab, sequences, window, masks, *a); }''')
    lib.rules.restype = C.c_char_p
    A = arrays("A", ["logits", "starts", "tokens", "history", "lengths", "penalties", "bias", "masks", "mask_of", "output"],
               ["lp", "hp", "bp", "mp", "op"])
    lib.rules.argtypes = [C.c_int] * 6 + [C.POINTER(A)]
    good = dict(dtype=2, rows=5, vocab=1000, sequences=2, window=0, mask_count=3)
    data = dict(logits=18, starts=20, tokens=24, history=32, lengths=36, penalties=40, bias=44, masks=48, mask_of=52, output=18, lp=1000,
                hp=0, bp=1000, mp=32, op=1000)

    def check(**kw):
        return lib.rules(*{k: kw.get(k, v) for k, v in good.items()}.values(), A(**{k: kw.get(k, v) for k, v in data.items()}))
    assert check() is None and check(bp=0) is None and check(rows=0, logits=None) is None and check(sequences=0, starts=None) is None
    assert check(tokens=None, history=None, lengths=None, penalties=None, bias=None, masks=None, mask_of=None, mask_count=-1) is None
    assert check(rows=65535, sequences=65535, vocab=1 << 28, lp=1 << 28, op=1 << 28, bp=0, mp=1 << 23, hp=1 << 30) is None
    for bad in (dict(dtype=3), dict(rows=65536), dict(rows=-1), dict(sequences=65536), dict(sequences=-1), dict(vocab=0),
                dict(vocab=(1 << 28) + 1), dict(window=-1), dict(logits=None), dict(output=None), dict(starts=None), dict(lengths=None),
                dict(mask_of=None), dict(logits=17), dict(output=17), dict(starts=18), dict(tokens=20), dict(history=36), dict(lengths=18),
                dict(penalties=18), dict(bias=18), dict(masks=18), dict(mask_of=18), dict(lp=999), dict(lp=1 << 32), dict(op=999),
                dict(hp=-1), dict(hp=(1 << 30) + 1), dict(bp=999), dict(bp=-1), dict(mask_count=-1), dict(mp=31), dict(mp=1 << 32),
                dict(lp=1001)):
        assert check(**bad), bad


def test_delta_rule_checks_and_bytes(tmp_path):
    lib = compiled(tmp_path, '''
#include "step_checks.h"
using namespace fortai_hip;
static GdnShape shape(const int *n) {
    GdnShape s; s.layers = n[0]; s.slots = n[1]; s.key_heads = n[2]; s.value_heads = n[3]; s.head = n[4]; s.taps = n[5]; s.pending = n[6];
    return s; }
extern "C" {
const char *cache(const int *n) { return check_gdn_shape(shape(n)); }
size_t bytes(const int *n) { return gdn_bytes(shape(n)); }
const char *rows(int n) { return check_gdn_rows(n); }
const char *batch(int sequences, int rows, int most_rows, int most, const void *starts, const void *slots, const void *standing) {
    return check_gdn_batch(sequences, rows, most_rows, most, starts, slots, standing); }
const char *run(const int *n, int layer, int dtype, int rows, float eps, const GdnArrays *a) {
    return check_gdn_run(shape(n), layer, dtype, rows, eps, *a); }
const char *pairs(const int32_t *from, const int32_t *to, int count, int slots) { return check_slot_pairs(from, to, count, slots); }
}''')
    for f in (lib.cache, lib.rows, lib.batch, lib.run, lib.pairs):
        f.restype = C.c_char_p
    lib.bytes.restype = C.c_size_t
    shape = dict(layers=2, slots=3, key_heads=2, value_heads=4, head=64, taps=4, pending=5)
    ints = lambda **kw: (C.c_int * 7)(*{**shape, **kw}.values())
    assert lib.cache(ints()) is None and lib.cache(ints(pending=0, taps=2, head=128)) is None
    for bad in (dict(layers=0), dict(layers=4097), dict(slots=0), dict(slots=-1), dict(key_heads=0), dict(value_heads=3),
                dict(value_heads=0), dict(key_heads=1025, value_heads=1025), dict(value_heads=2048), dict(head=32), dict(head=256),
                dict(taps=1), dict(taps=9), dict(pending=-1), dict(pending=17)):
        assert lib.cache(ints(**bad)) and lib.bytes(ints(**bad)) == 0, bad
    rng = random.Random(4)
    for _ in range(300):
        kh = rng.choice([1, 3, 16, 1024])
        kw = dict(layers=rng.choice([1, 7, 4096]), slots=rng.choice([1, 9, 1 << 20, (1 << 31) - 1]), key_heads=kh,
                  value_heads=kh * (1 if kh == 1024 else rng.choice([1, 4])), head=rng.choice([64, 128]), taps=rng.randint(2, 8),
                  pending=rng.randint(0, 16))
        d, vh, p = kw["head"], kw["value_heads"], kw["pending"]
        want = kw["layers"] * kw["slots"] * 4 * (vh * d * d + (kw["taps"] - 1 + p) * (2 * kh + vh) * d + p * (kh * d + vh * d + vh) + 1)
        got = lib.bytes(ints(**kw))
        assert got == want if want < 8.9e15 else got == 0 or got == want, kw
        if want < 8.9e15:
            assert B.load().fortai_hip_gdn_bytes(*kw.values()) == want
    assert lib.rows(1) is None and lib.rows(1 << 19) is None and lib.rows(0) and lib.rows((1 << 19) + 1)
    good = dict(sequences=3, rows=20, most_rows=9, most=64, starts=20, slots=24, standing=None)
    lib.batch.argtypes = [C.c_int] * 4 + [C.c_void_p] * 3
    batch = lambda **kw: lib.batch(*{**good, **kw}.values())
    assert batch() is None and batch(standing=28) is None and batch(rows=0, most_rows=0, starts=None) is None
    assert batch(sequences=0, slots=None) is None and batch(rows=64) is None
    for bad in (dict(sequences=-1), dict(sequences=16385), dict(rows=-1, most_rows=0), dict(rows=65), dict(most_rows=21), dict(most_rows=-1),
                dict(starts=None), dict(slots=None), dict(starts=18), dict(slots=18), dict(standing=18)):
        assert batch(**bad), bad
    A = arrays("A", ["qkv", "alpha", "beta", "conv", "a", "dt", "output"], ["qp", "ap", "bp", "op"])
    lib.run.argtypes = [C.c_void_p] + [C.c_int] * 3 + [C.c_float, C.POINTER(A)]
    call = dict(layer=1, dtype=1, rows=2, eps=1e-6)
    data = dict(qkv=18, alpha=18, beta=18, conv=20, a=20, dt=20, output=18, qp=0, ap=0, bp=0, op=256)

    def run(**kw):
        return lib.run(ints(), *{k: kw.get(k, v) for k, v in call.items()}.values(), A(**{k: kw.get(k, v) for k, v in data.items()}))
    assert run() is None and run(rows=1, op=0) is None
    for bad in (dict(layer=2), dict(layer=-1), dict(dtype=3), dict(eps=0.0), dict(eps=NAN), *({n: None} for n in list(data)[:7]),
                *({n: 17} for n in list(data)[:7]), dict(conv=18), dict(a=18), dict(dt=18), dict(qp=-1), dict(ap=1 << 32), dict(bp=-1),
                dict(op=255), dict(op=1 << 32)):
        assert run(**bad), bad
    array = lambda *n: (C.c_int32 * len(n))(*n)
    assert lib.pairs(array(0, 0), array(1, 2), 2, 3) is None
    for f, t in (((0, 1), (2, 2)), ((0, 1), (1, 2)), ((3,), (0,)), ((0,), (-1,)), ((1,), (1,))):
        assert lib.pairs(array(*f), array(*t), len(f), 3), (f, t)


def test_group_checks_and_plan(tmp_path):
    lib = compiled(tmp_path, '''
#include "kv8_device.h"
#include "serving_checks.h"
using namespace fortai_hip;
extern "C" {
const char *check(int groups, int most, int rows, int sequences, int shared, const void *starts, const void *s, const void *of) {
    return check_kv8_groups(groups, most, rows, sequences, shared, starts, s, of); }
void plan(int fp32, int head, int sequences, int groups, int kv, int64_t rows, int64_t group_rows, int64_t own, int64_t shared, int64_t *out) {
    const Kv8SharedPlan p = kv8_shared_plan(fp32 != 0, head, sequences, groups, kv, rows, group_rows, own, shared);
    const int64_t all[] = {p.shares, p.own_at, p.own.rows, p.own.row_tiles, p.own.splits, p.group.rows, p.group.row_tiles, p.group.splits,
        kKv8SharedRows, kKv8MaxSplits};
    for (int i = 0; i < 10; ++i) out[i] = all[i]; }
}''')
    lib.check.restype = C.c_char_p
    lib.check.argtypes = [C.c_int] * 5 + [C.c_void_p] * 3
    good = dict(groups=2, most=7, rows=9, sequences=5, shared=100, starts=20, s=24, of=28)
    check = lambda **kw: lib.check(*{**good, **kw}.values())
    assert check() is None and check(groups=0, starts=None, s=None, of=None) is None and check(groups=5, most=0, shared=0) is None
    for bad in (dict(groups=-1), dict(groups=6), dict(most=-1), dict(most=10), dict(shared=-1), dict(starts=None), dict(s=None),
                dict(of=None), dict(starts=18), dict(s=18), dict(of=18)):
        assert check(**bad), bad
    lib.plan.argtypes = [C.c_int] * 5 + [C.c_int64] * 4 + [C.c_void_p]
    out, rng, shared_ones = (C.c_int64 * 10)(), random.Random(2), 0
    for _ in range(4000):
        sequences = rng.choice([1, 2, 8, 37, 1000, 16384])
        groups, rows = rng.randint(1, sequences), int(2 ** rng.uniform(0, 12))
        group_rows = max(1, int(rows * rng.uniform(1, sequences)))
        kv = rng.choice([1, 2, 4, 8, 64])
        own, shared = int(2 ** rng.uniform(0, 20)) - 1, int(2 ** rng.uniform(0, 30)) - 1
        lib.plan(rng.randrange(2), rng.choice([64, 128, 256]), sequences, groups, kv, rows, group_rows, own, shared, out)
        shares, own_at, own_rows, own_tiles, own_splits, tile, tiles, splits, room, most = out[:]
        shared_ones += shares
        assert own_at % 64 == 0 and 1 <= splits <= most and 1 <= own_splits <= most
        assert tiles * tile >= group_rows and own_tiles * own_rows >= rows
        if shares:  # every partial result has its place, the groups' before the sequences'
            assert shared >= 64 and groups * tiles * kv * tile * splits <= own_at
            assert own_at + sequences * own_tiles * kv * own_rows * own_splits <= room
    assert shared_ones > 200


def model_groups(tables, lengths, page):
    """The groups as their rule says it: the ones that follow join while 64 tokens or more are common and reading those once saves more."""
    common = lambda a, b: min(len(list(itertools.takewhile(lambda p: p[0] == p[1] >= 0, zip(tables[a], tables[b])))) * page, lengths[b])
    groups, first = [], 0
    while first < len(tables):
        end, tokens = first + 1, lengths[first]
        while end < len(tables):
            t, members = min(common(first, end), tokens), end - first
            if t < 64 or (members > 1 and t * members < tokens * (members - 1)):
                break
            tokens, end = t, end + 1
        groups.append((first, end, tokens if end > first + 1 else 0))
        first = end
    merged = []
    for g in groups:
        if merged and g[2] == 0 == merged[-1][2]:
            merged[-1] = (merged[-1][0], g[1], 0)
        else:
            merged.append(g)
    return merged


@pytest.mark.parametrize("seed", range(6))
def test_groups_against_a_model(seed):
    rng = random.Random(seed)
    page = rng.choice([16, 32, 64])
    pool = B.Kv8Pages(600, page, 12, 40)
    some = 0
    try:
        for _ in range(800):
            seq, kind = rng.randrange(12), rng.random()
            try:
                if kind < 0.4:
                    pool.extend(seq, rng.randint(1, 4 * page))
                elif kind < 0.85:
                    other = rng.randrange(12)
                    if pool.length(seq) == 0 and pool.length(other) > 0:
                        pool.fork(other, seq, rng.choice([pool.length(other), rng.randint(1, pool.length(other))]))
                else:
                    pool.truncate(seq, rng.choice([0, rng.randint(0, pool.length(seq))]))
            except B.BackendError:
                pass  # no pages left
            who = rng.sample(range(12), rng.randint(0, 12))
            if rng.random() < 0.5:
                who.sort()
            starts, shared, group_of = pool.groups(who)
            want = model_groups([pool.tables([s])[0].tolist() for s in who], [pool.length(s) for s in who], page)
            some += any(w[2] for w in want)
            assert starts.tolist() == [w[0] for w in want] + [len(who)] and shared.tolist() == [w[2] for w in want]
            assert group_of.tolist() == [g for g, w in enumerate(want) for _ in range(w[0], w[1])]
    finally:
        pool.free()
    assert some > 10  # there was something to find


def test_groups_refusals():
    pool = B.Kv8Pages(8, 16, 2, 4)
    lib, n = B.load(), C.c_int(7)
    try:
        one = lambda: np.zeros(3, dtype=np.int32)
        starts, shared, of, who = one(), one(), one(), one()
        at = lambda a: a.ctypes.data
        f = lib.fortai_hip_kv8_pages_groups
        assert f(pool.h, at(who), 0, at(starts), None, None, C.byref(n)) == 0 and n.value == 0 and starts[0] == 0
        who[0] = 2
        with pytest.raises(B.BackendError):
            pool.groups([0, 2])
        for args in ((None, at(who), 1, at(starts), at(shared), at(of), C.byref(n)), (pool.h, None, 1, at(starts), at(shared), at(of), C.byref(n)),
                     (pool.h, at(who), -1, at(starts), at(shared), at(of), C.byref(n)), (pool.h, at(who), 1, None, at(shared), at(of), C.byref(n)),
                     (pool.h, at(who), 1, at(starts), None, at(of), C.byref(n)), (pool.h, at(who), 1, at(starts), at(shared), None, C.byref(n)),
                     (pool.h, at(who), 1, at(starts), at(shared), at(of), None)):
            assert f(*args) != 0
    finally:
        pool.free()


def test_calls_without_a_handle_are_refused():
    lib = B.load()
    batch, rules, groups = B.GdnBatch(0, 0, 0, 16, 16), B.LogitRules(), B.Kv8Groups(0, 0, 16, 16, 16)
    assert lib.fortai_hip_norm_tokens_device(None, 0, 16, 32, None, 0, None, 0, None, 32, 1.0, None, 0, 1, 32, 16, 32, None) != 0
    assert lib.fortai_hip_q8_tokens_read_device(None, 0, 16, 1, 32, 16, 32) != 0
    assert lib.fortai_hip_logits_adjust_device(None, 0, 16, 8, 1, 8, 1, 16, C.byref(rules), 16, 8) != 0
    assert lib.fortai_hip_gdn_run_device(None, 0, C.byref(batch), 0, 16, 0, 16, 0, 16, 0, 16, 16, 16, 1.0, 16, 64) != 0
    assert lib.fortai_hip_gdn_copy_slots(None, None, None, 0) != 0 and lib.fortai_hip_gdn_destroy(None) == 0
    assert lib.fortai_hip_kv8_shared_attention_device(None, 0, None, C.byref(groups), 0, 16, 0, 0, None, 1, 1.0, 1, 1, 16, 64) != 0
