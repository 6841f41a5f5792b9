"""The operators of a serving step over a shared 8-bit cache, and their plain forms.

A server that decodes several sequences with drafted tokens rotates the new
queries and keys, stores keys and values in an 8-bit paged cache, attends over
it, copies pages when sequences fork or the pool is compacted, and decides
which drafts stand.  Each case is one of those calls at one size; ``draw``
gives further sizes of the same ranges.  With ``own`` false ``run`` computes
the same results in elementary torch operations.

Head layouts are those of ``fortai_amd.synth.CONFIGS`` (8 / 2, 16 / 4 and 4 / 2
heads of 256 and 64) and generic ones; sequences of a batch differ in length.
"""

import math

import numpy as np
import torch

if torch.cuda.is_available():
    DEV = "cuda"
else:
    DEV = "cpu"

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------- cases
def listed():
    return [
        # the smallest call: q and k heads of one decode step of eight sequences, normalised and rotated
        {"name": "rope_decode", "kind": "rope", "rows": 8, "heads": 20, "head": 256, "rotary": 64,
         "interleaved": False, "norm": True, "scaling": "none", "far": 8000, "dtype": "f32"},
        # a prompt block at the far end of a stretched context
        {"name": "rope_prompt", "kind": "rope", "rows": 4096, "heads": 20, "head": 128, "rotary": 128,
         "interleaved": True, "norm": False, "scaling": "yarn", "far": 500000, "dtype": "bf16"},
        # one new token of each of eight sequences
        {"name": "append_decode", "kind": "append", "kv_heads": 4, "head": 256, "page": 64, "sequences": 8, "rows": 1,
         "length": 8000, "dtype": "f32"},
        # eight prompts of up to 512 tokens, each behind a cached prefix that ends inside a page
        {"name": "append_prompt", "kind": "append", "kv_heads": 4, "head": 256, "page": 64, "sequences": 8,
         "rows": 512, "length": 777, "dtype": "bf16"},
        # one sequence early in a conversation
        {"name": "attention_short", "kind": "attention", "heads": 8, "kv_heads": 2, "head": 256, "page": 32,
         "sequences": 1, "rows": 1, "length": 600, "gate": True, "dtype": "f32"},
        # a decode step of eight sequences of unlike lengths, up to a context of 8192
        {"name": "attention_batch", "kind": "attention", "heads": 16, "kv_heads": 4, "head": 256, "page": 64,
         "sequences": 8, "rows": 1, "length": 8190, "gate": True, "dtype": "f32"},
        # four drafts and the token before them, deep in one long document
        {"name": "attention_drafts", "kind": "attention", "heads": 8, "kv_heads": 2, "head": 256, "page": 64,
         "sequences": 1, "rows": 5, "length": 32760, "gate": True, "dtype": "bf16"},
        # a chunk of a prompt behind the chunks that are cached already
        {"name": "attention_prompt", "kind": "attention", "heads": 16, "kv_heads": 4, "head": 256, "page": 64,
         "sequences": 1, "rows": 2000, "length": 6000, "gate": False, "dtype": "bf16"},
        # a sequence forks: its last, partly filled page in each of eight layers
        {"name": "pages_fork", "kind": "pages", "layers": 8, "kv_heads": 4, "head": 256, "page": 64, "pages": 64,
         "copies": 1},
        # a fragmented pool is compacted
        {"name": "pages_compact", "kind": "pages", "layers": 8, "kv_heads": 4, "head": 256, "page": 64, "pages": 1200,
         "copies": 500},
        # four drafts of one sequence without draft probabilities (looked up in the text), a small vocabulary
        {"name": "verify_lookup", "kind": "verify", "sequences": 1, "rows": 5, "vocab": 16384, "drafts": False,
         "masked": False, "greedy": False, "dtype": "f32"},
        # up to four drafts of each of eight sequences, against a draft model's logits
        {"name": "verify_batch", "kind": "verify", "sequences": 8, "rows": 5, "vocab": 248320, "drafts": True,
         "masked": True, "greedy": True, "dtype": "f32"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "attention", "attention", "attention", "pages", "verify"])
    heads, kv_heads = rng.choice([(8, 2), (16, 4), (4, 2), (6, 6), (12, 1), (5, 5), (24, 3)])
    head = rng.choice([64, 128, 256])
    page = rng.choice([16, 32, 64])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "rope":
        return {"kind": kind, "rows": _log(rng, 1, 4096), "heads": rng.randint(1, 20), "head": head,
                "rotary": rng.choice([head, head // 2, head // 4, 2 * rng.randint(1, head // 2)]),
                "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "yarn"]), "far": _log(rng, 10, 1000000), "dtype": dtype}
    if kind == "append":
        sequences = rng.randint(1, 8)
        return {"kind": kind, "kv_heads": kv_heads, "head": head, "page": page, "sequences": sequences,
                "rows": _log(rng, 1, 4096 // sequences), "length": _log(rng, 1, 8000), "dtype": dtype}
    if kind == "attention":
        form = rng.choice(["decode", "decode", "drafts", "chunk"])
        sequences = rng.randint(1, 8)
        case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "head": head, "page": page, "sequences": sequences,
                "rows": 1, "length": _log(rng, 1, 32760 // sequences), "gate": rng.random() < 0.5, "dtype": dtype}
        if form == "drafts":
            case["rows"] = rng.randint(2, 17)
        elif form == "chunk":
            case["sequences"] = rng.randint(1, 3)
            case["rows"] = _log(rng, 18, 1500 // case["sequences"])
            case["length"] = _log(rng, 1, 6000 // case["sequences"])
        return case
    if kind == "pages":
        copies = _log(rng, 1, 500)
        return {"kind": kind, "layers": rng.randint(1, 8), "kv_heads": min(kv_heads, 4), "head": head, "page": page,
                "pages": 2 * copies + rng.randint(0, 60), "copies": copies}
    return {"kind": kind, "sequences": rng.randint(1, 8), "rows": rng.randint(1, 5),
            "vocab": rng.choice([4096, 16384, 248320, _log(rng, 500, 240000)]), "drafts": rng.random() < 0.6,
            "masked": rng.random() < 0.5, "greedy": rng.random() < 0.5, "dtype": dtype}


def _lengths(case):
    """Cached tokens and new rows of each sequence: the first has the most, later ones down to a fifth."""
    n, length, rows = case["sequences"], case["length"], case["rows"]
    share = [1.0 - 0.8 * s / max(1, n - 1) if s else 1.0 for s in range(n)]
    return [max(0, int(length * f)) for f in share], [max(1, int(round(rows * (1.0 - 0.37 * (s % 3) / 2)))) for s in range(n)]


def _verify_rows(case):
    return [max(1, case["rows"] - (s % 3)) for s in range(case["sequences"])]


# ------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(0x0B5E + 6151 * int(seed))
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


_CONTEXT = None


def _context():
    """The program's one context: its calls run in order on one stream."""
    global _CONTEXT
    if _CONTEXT is None:
        from fortai_amd import backend
        _CONTEXT = backend.Context(0)
    return _CONTEXT


class _State:
    """What a program holds for one case; its handles are given back with it."""

    def __init__(self, case):
        self.case = case
        self.handles = []

    def __del__(self):
        try:
            for h in self.handles:
                h.free()
        except Exception:
            pass


def _storage(g, layers, pages, kv_heads, page, head):
    """A filled cache: key codes [layers][pages][kv_heads][page][head], value codes
    [layers][pages][kv_heads][head][page], then the maxima of each page and head, keys' and values'."""
    n = layers * pages * kv_heads
    codes, scales = n * page * head, 4 * n
    storage = torch.empty(2 * codes + 2 * scales, dtype=torch.uint8, device=DEV)
    step = 1 << 26
    for at in range(0, 2 * codes, step):
        m = min(step, 2 * codes - at)
        storage[at:at + m] = (_normal(g, m) * 36.0).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    maxima = torch.exp(0.25 * _normal(g, 2 * n)) * 3.5
    storage[2 * codes:] = maxima.view(torch.uint8)
    return storage


def _planes(storage, layers, pages, kv_heads, page, head):
    """The storage's four planes, as views."""
    n = layers * pages * kv_heads
    codes = n * page * head
    keys = storage[:codes].view(torch.int8).view(layers, pages, kv_heads, page, head)
    values = storage[codes:2 * codes].view(torch.int8).view(layers, pages, kv_heads, head, page)
    maxima = storage[2 * codes:].view(torch.float32).view(2, layers, pages, kv_heads)
    return keys, values, maxima[0], maxima[1]


def _cache_inputs(s, g, case, spare):
    """Storage of one layer, page tables in a shuffled order, and the sequences' lengths."""
    lengths, rows = _lengths(case)
    page = case["page"]
    need = [-(-(l + r) // page) for l, r in zip(lengths, rows)]
    s.pages, s.pitch = sum(need) + spare, max(need)
    order = torch.randperm(s.pages, generator=g, device=DEV).to(torch.int32)
    tables = torch.full((len(need), s.pitch), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, k in enumerate(need):
        tables[i, :k] = order[at:at + k]
        at += k
    s.tables = tables
    s.storage = _storage(g, 1, s.pages, case["kv_heads"], page, case["head"])
    s.total, s.most, s.longest = sum(rows), max(rows), max(l + r for l, r in zip(lengths, rows))
    s.row_starts = _int32(np.concatenate([[0], np.cumsum(rows)]).tolist())
    s.lengths = _int32(lengths)
    s.host_lengths, s.host_rows = lengths, rows


# ----------------------------------------------------------------- prepare
def prepare(case, seed):
    s = _State(case)
    globals()["_prepare_" + case["kind"]](s, _generator(seed), case)
    if own:
        _hold(s, case)
    if DEV == "cuda":
        torch.cuda.synchronize()
    return s


def _hold(s, case):
    """The framework's handles over these inputs, which a program keeps beside them (the inputs are the same without)."""
    from fortai_amd import backend
    kind, ctx = case["kind"], _context()
    if kind == "rope":
        base, (factor, original, fast, slow, attention) = _rope_numbers(case)
        s.handles.append(backend.Rope(
            ctx, case["rotary"], interleaved=case["interleaved"], base=base, scaling=case["scaling"], factor=factor,
            original_context=original, beta_fast=fast, beta_slow=slow, attention_factor=attention))
    elif kind == "verify":
        s.handles.append(backend.Verifier(ctx, s.total, case["sequences"], case["vocab"]))
    else:
        s.handles.append(backend.Kv8Cache(
            ctx, case.get("layers", 1), case["pages"] if kind == "pages" else s.pages, case["page"], case["kv_heads"],
            case["head"], storage=s.storage.data_ptr(), storage_bytes=s.storage.numel()))
    if kind in ("append", "attention"):
        s.batch = backend.Kv8Batch(case["sequences"], s.total, s.most, s.row_starts.data_ptr(), s.lengths.data_ptr(),
                                   s.tables.data_ptr(), s.pitch)
    if kind == "append":
        s.again = backend.Kv8Batch(case["sequences"], s.read_total, s.read_most, s.read_starts.data_ptr(),
                                   s.read_first.data_ptr(), s.tables.data_ptr(), s.pitch)


def _rope_numbers(case):
    """base, scaling and its numbers (factor, original context, fast, slow, attention factor)."""
    if case["scaling"] == "none":
        return 1.0e7, (1.0, 0, 32.0, 1.0, 1.0)
    if case["scaling"] == "linear":
        return 1.0e4, (8.0, 0, 32.0, 1.0, 1.0)
    return 1.0e6, (16.0, 32768, 32.0, 1.0, 0.1 * math.log(16.0) + 1.0)


def _prepare_rope(s, g, case):
    rows, heads, head, dtype = case["rows"], case["heads"], case["head"], DTYPES[case["dtype"]]
    s.x = _normal(g, rows, heads, head).to(dtype)
    s.weight = 1.0 + 0.1 * _normal(g, head) if case["norm"] else None
    first = int(torch.randint(0, case["far"], (1,), generator=g, device=DEV))
    s.positions = (first + torch.arange(rows, device=DEV)).to(torch.int32)
    s.out = torch.empty_like(s.x)


def _prepare_append(s, g, case):
    _cache_inputs(s, g, case, 5)
    kv, head, dtype = case["kv_heads"], case["head"], DTYPES[case["dtype"]]
    # the rows of one projection's output: keys and values side by side
    loud = torch.exp(0.3 * _normal(g, 1, 2, kv, 1))
    s.kv = (_normal(g, s.total, 2, kv, head) * loud * 1.2).to(dtype)
    # read back from the start of the page that the first new token falls into
    page = case["page"]
    first = [l // page * page for l in s.host_lengths]
    counts = [l + r - f for l, r, f in zip(s.host_lengths, s.host_rows, first)]
    s.read_first, s.read_starts = _int32(first), _int32(np.concatenate([[0], np.cumsum(counts)]).tolist())
    s.read_total, s.read_most = sum(counts), max(counts)
    s.keys = torch.empty(s.read_total, kv, head, dtype=torch.float32, device=DEV)
    s.values = torch.empty_like(s.keys)


def _prepare_attention(s, g, case):
    _cache_inputs(s, g, case, 3)
    heads, head, dtype = case["heads"], case["head"], DTYPES[case["dtype"]]
    parts = 2 if case["gate"] else 1
    q = _normal(g, s.total, heads, parts, head)
    q[:, :, 0] *= 2.0 * torch.exp(0.3 * _normal(g, 1, heads, 1))
    s.q = q.to(dtype)
    s.scale = 1.0 / math.sqrt(head)
    s.out = torch.empty(s.total, heads, head, dtype=dtype, device=DEV)


def _prepare_pages(s, g, case):
    s.storage = _storage(g, case["layers"], case["pages"], case["kv_heads"], case["page"], case["head"])
    order = torch.randperm(case["pages"], generator=g, device=DEV).cpu().numpy().astype(np.int32)
    n = case["copies"]
    # as a compaction: live pages from the upper end into the lower end's holes
    chosen = np.sort(order[:2 * n])
    s.to, s.source = np.ascontiguousarray(chosen[:n]), np.ascontiguousarray(chosen[n:])
    s.device_to, s.device_source = (torch.from_numpy(a).to(DEV).long() for a in (s.to, s.source))


def _prepare_verify(s, g, case):
    rows, vocab, dtype = _verify_rows(case), case["vocab"], DTYPES[case["dtype"]]
    s.total, s.most = sum(rows), max(rows)
    target = 2.5 * _normal(g, s.total, vocab)
    if case["masked"]:
        target[:, torch.rand(vocab, generator=g, device=DEV) < 0.1] = -math.inf
    noise = -torch.log(-torch.log(torch.rand(s.total, vocab, generator=g, device=DEV).clamp(1e-20, 1 - 1e-7)))
    if case["drafts"]:
        s.draft = (target + 0.4 * _normal(g, s.total, vocab)).to(dtype)
        chosen = (s.draft.float() + noise).argmax(dim=1)
    else:
        s.draft = None
        chosen = (1.5 * target + 0.5 * noise).argmax(dim=1)
    s.target = target.to(dtype)
    # row r + 1 of the step was fed the draft that row r's distribution gave
    s.tokens = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), chosen[:-1]])
    s.uniforms = torch.rand(s.total, generator=g, device=DEV)
    s.temperatures = 0.5 + torch.rand(case["sequences"], generator=g, device=DEV)
    if case["greedy"]:
        s.temperatures[1::3] = 0.0
    s.row_starts = _int32(np.concatenate([[0], np.cumsum(rows)]).tolist())
    s.emitted = torch.empty(s.total, dtype=torch.int64, device=DEV)
    s.accepted = torch.empty(case["sequences"], dtype=torch.int32, device=DEV)
    s.logprobs = torch.empty(s.total, dtype=torch.float32, device=DEV)


# --------------------------------------------------------------------- run
def run(state):
    return globals()[("_own_" if own else "_run_") + state.case["kind"]](state, state.case)


def _own_rope(s, case):
    s.handles[0].apply(s.x.data_ptr(), s.positions.data_ptr(), case["rows"], case["heads"], case["head"],
                       s.out.data_ptr(), dtype=case["dtype"], norm=None if s.weight is None else s.weight.data_ptr(),
                       eps=1e-6)
    return s.out


def _own_append(s, case):
    cache, width, at = s.handles[0], case["kv_heads"] * case["head"], s.kv.data_ptr()
    cache.append(0, s.batch, at, at + width * s.kv.element_size(), dtype=case["dtype"], key_pitch=2 * width,
                 value_pitch=2 * width)
    cache.read(0, s.again, s.keys.data_ptr(), s.values.data_ptr(), dtype="f32")
    return {"keys": s.keys, "values": s.values}


def _own_attention(s, case):
    parts, head, at = s.q.shape[2], case["head"], s.q.data_ptr()
    s.handles[0].attention(0, s.batch, at, case["heads"], s.out.data_ptr(), s.scale, s.longest, dtype=case["dtype"],
                           gate=at + head * s.q.element_size() if parts == 2 else None, query_head_pitch=parts * head,
                           query_pitch=case["heads"] * parts * head)
    return s.out


def _own_pages(s, case):
    s.handles[0].copy_pages(s.source, s.to)
    return s.storage


def _own_verify(s, case):
    s.handles[0].run(s.target.data_ptr(), s.tokens.data_ptr(), s.uniforms.data_ptr(), s.row_starts.data_ptr(),
                     case["sequences"], s.total, s.emitted.data_ptr(), s.accepted.data_ptr(), dtype=case["dtype"],
                     draft_logits=None if s.draft is None else s.draft.data_ptr(),
                     temperatures=s.temperatures.data_ptr(), logprobs=s.logprobs.data_ptr())
    return {"tokens": s.emitted, "accepted": s.accepted, "logprobs": s.logprobs}


# ------------------------------------------------------------- plain forms
def _frequencies(case):
    """Turns' angle of each pair for one position, in 64 bits."""
    r = case["rotary"]
    base, (factor, original, fast, slow, attention) = _rope_numbers(case)
    i = torch.arange(0, r, 2, dtype=torch.float64, device=DEV)
    theta = torch.pow(torch.tensor(base, dtype=torch.float64, device=DEV), -i / r)
    if case["scaling"] == "linear":
        theta = theta / factor
    if case["scaling"] == "yarn":
        # the pair that makes this many turns within the original context
        pair = lambda turns: r * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))
        low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), r - 1)
        ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0.0, 1.0)
        theta = theta / factor * ramp + theta * (1.0 - ramp)
    return theta, attention


def _run_rope(s, case):
    r = case["rotary"]
    x = s.x.float()
    if s.weight is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + 1e-6) * s.weight
    theta, attention = _frequencies(case)
    angle = s.positions.double()[:, None, None] * theta
    c, w = (torch.cos(angle) * attention).float(), (torch.sin(angle) * attention).float()
    out = x.clone()
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        out[..., 0:r:2], out[..., 1:r:2] = a * c - b * w, a * w + b * c
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        out[..., :r // 2], out[..., r // 2:r] = a * c - b * w, a * w + b * c
    return out.to(s.x.dtype)


def _padded(starts, most):
    """Row numbers [sequences][most] of a ragged batch, and which of them are there."""
    starts = starts.long()
    t = torch.arange(most, device=DEV)
    rows = starts[:-1, None] + t
    there = rows < starts[1:, None]
    return torch.where(there, rows, torch.zeros_like(rows)), there


def _quantized(values, maxima):
    """codes = 127 x / maximum rounded half to even; in 64 bits, where the quotient of two
    such values next to a half stays on its side."""
    m = maxima.double()
    return torch.where(m > 0, torch.round(values.double() * 127.0 / m), torch.zeros_like(m)).clamp(-127, 127)


def _requantized(codes, old, new):
    return torch.where(new > old, torch.round(codes.double() * old.double() / new.double().clamp_min(1e-300)),
                       codes.double())


def _run_append(s, case):
    page, kv, head = case["page"], case["kv_heads"], case["head"]
    keys, values, key_max, value_max = (p[0] for p in _planes(s.storage, 1, s.pages, kv, page, head))
    first = s.lengths.long() // page
    span = (s.most + page - 1) // page + 1
    # every page that may be touched, and for each of its slots the new row that goes there
    slot_page = first[:, None] + torch.arange(span, device=DEV)
    token = slot_page[:, :, None] * page + torch.arange(page, device=DEV)
    row = token - s.lengths.long()[:, None, None]
    count = (s.row_starts[1:] - s.row_starts[:-1]).long()
    new = (row >= 0) & (row < count[:, None, None])
    seq, j = torch.nonzero(new.any(dim=2), as_tuple=True)
    ids = s.tables[seq, slot_page[seq, j]].long()
    row, new, token = row[seq, j], new[seq, j], token[seq, j]
    old = token < s.lengths.long()[seq][:, None]
    source = (s.row_starts[:-1].long()[seq][:, None] + row).clamp(0, s.total - 1)
    x = s.kv.float()[source]                                        # [touched][page][2][kv][head]
    x = torch.where(new[:, :, None, None, None], x, torch.zeros_like(x))
    some_old = old.any(dim=1)
    for plane, maxima, part in ((keys, key_max, 0), (values, value_max, 1)):
        v = x[:, :, part].transpose(1, 2)                           # [touched][kv][page][head]
        was = torch.where(some_old[:, None], maxima[ids], torch.zeros_like(maxima[ids]))
        now = torch.maximum(was, v.abs().amax(dim=(2, 3)))
        codes = plane[ids] if part == 0 else plane[ids].transpose(2, 3)
        kept = _requantized(codes, was[:, :, None, None], now[:, :, None, None])
        fresh = _quantized(v, now[:, :, None, None].expand_as(v))
        mixed = torch.where(new[:, None, :, None], fresh,
                            torch.where(old[:, None, :, None], kept, codes.double())).to(torch.int8)
        plane[ids] = mixed if part == 0 else mixed.transpose(2, 3).contiguous()
        maxima[ids] = now
    # read back
    rows, there = _padded(s.read_starts, s.read_most)
    token = s.read_first.long()[:, None] + torch.arange(s.read_most, device=DEV)
    token = torch.where(there, token, torch.zeros_like(token))
    ids = torch.gather(s.tables.long(), 1, token // page)[there]
    slot = (token % page)[there]
    k = keys[ids, :, slot].float() * (key_max[ids] / 127.0)[:, :, None]
    v = values[ids, :, :, slot].float() * (value_max[ids] / 127.0)[:, :, None]
    return {"keys": k, "values": v}


def _run_attention(s, case):
    page, kv, head, heads, n = case["page"], case["kv_heads"], case["head"], case["heads"], case["sequences"]
    keys, values, key_max, value_max = (p[0] for p in _planes(s.storage, 1, s.pages, kv, page, head))
    ids = s.tables.long().clamp_min(0)
    k = (keys[ids].float() * (key_max[ids] / 127.0)[..., None, None]).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, head)
    v = (values[ids].float() * (value_max[ids] / 127.0)[..., None, None]).permute(0, 2, 1, 4, 3).reshape(n, kv, -1, head)
    rows, there = _padded(s.row_starts, s.most)
    q = s.q[:, :, 0].float()[rows]                                  # [n][most][heads][head]
    group = heads // kv
    q = q.reshape(n, s.most, kv, group, head).permute(0, 2, 3, 1, 4).reshape(n, kv, group * s.most, head)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) * s.scale
    scores = scores.reshape(n, kv, group, s.most, -1)
    position = s.lengths.long()[:, None] + torch.arange(s.most, device=DEV)
    seen = torch.arange(scores.shape[-1], device=DEV) <= position[:, None, None, :, None]
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - top)
    p = p / p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p.reshape(n, kv, group * s.most, -1), v)
    out = out.reshape(n, kv, group, s.most, head).permute(0, 3, 1, 2, 4).reshape(n, s.most, heads, head)[there]
    if case["gate"]:
        out = out / (1.0 + torch.exp(-s.q[:, :, 1].float()))
    return out.to(s.q.dtype)


def _run_pages(s, case):
    for plane in _planes(s.storage, case["layers"], case["pages"], case["kv_heads"], case["page"], case["head"]):
        plane[:, s.device_to] = plane[:, s.device_source]
    return s.storage


def _softmax64(logits, temperatures):
    """exp((l - max) / T) normalised, the maxima's logits, in 64 bits; T <= 0 counts as 1."""
    x = logits.double()
    t = temperatures.double()
    t = torch.where(t > 0, t, torch.ones_like(t))
    top = x.amax(dim=-1, keepdim=True)
    w = torch.exp((x - top) / t)
    return w / w.sum(dim=-1, keepdim=True)


def _run_verify(s, case):
    n, vocab, most = case["sequences"], case["vocab"], s.most
    rows, there = _padded(s.row_starts, most)
    drafts = there.sum(dim=1) - 1
    i = torch.arange(most, device=DEV)
    is_draft = i < drafts[:, None]
    greedy = s.temperatures <= 0
    p = _softmax64(s.target[rows], s.temperatures[:, None, None])   # [n][most][vocab]
    token = torch.arange(vocab, device=DEV)
    best = torch.where(p == p.amax(dim=-1, keepdim=True), token, torch.full_like(token, vocab)).amin(dim=-1)
    x = s.tokens[(rows + 1).clamp_max(s.total - 1)]
    if s.draft is None:
        q = (token == x[:, :, None]).double()
    else:
        q = _softmax64(s.draft[rows], s.temperatures[:, None, None])
    px, qx = torch.gather(p, 2, x[:, :, None])[..., 0], torch.gather(q, 2, x[:, :, None])[..., 0]
    stands = torch.where(greedy[:, None], x == best, s.uniforms.double()[rows] * qx < px) & is_draft
    accepted = torch.cumprod(stands.long(), dim=1).sum(dim=1)
    each = torch.arange(n, device=DEV)
    pa, qa = p[each, accepted], q[each, accepted]
    left = torch.where((accepted < drafts)[:, None], (pa - qa).clamp_min(0.0), pa)
    left = torch.where(left.sum(dim=1, keepdim=True) > 0, left, pa)
    c = torch.cumsum(left, dim=1)
    u = s.uniforms.double()[s.row_starts[1:].long() - 1]
    over = (c > (u * c[:, -1])[:, None]) & (left > 0)
    last = torch.where(left > 0, token, torch.zeros_like(token)).amax(dim=1)
    sampled = torch.minimum(torch.where(over, token, torch.full_like(token, vocab)).amin(dim=1), last)
    sampled = torch.where(greedy, best[each, accepted], sampled)
    out = torch.where(i < accepted[:, None], x, torch.where(i == accepted[:, None], sampled[:, None], torch.full_like(x, -1)))
    logp = torch.log(torch.gather(p, 2, out.clamp_min(0)[:, :, None])[..., 0])
    logp = torch.where(out >= 0, logp, torch.zeros_like(logp))
    return {"tokens": out[there], "accepted": accepted.to(torch.int32), "logprobs": logp.float()[there]}


# -------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    size = {"f32": 4, "f16": 2, "bf16": 2}[case.get("dtype", "f32")]
    if kind == "rope":
        n = case["rows"] * case["heads"] * case["head"]
        return {"bytes": 2 * n * size + 4 * case["rows"], "flops": n * (3 + (4 if case["norm"] else 0))}
    if kind == "pages":
        n = case["layers"] * case["copies"] * case["kv_heads"] * (2 * case["page"] * case["head"] + 8)
        return {"bytes": 2 * n, "flops": 0}
    if kind == "verify":
        rows = _verify_rows(case)
        total = sum(rows) + ((sum(rows) - case["sequences"]) if case["drafts"] else 0)
        return {"bytes": total * case["vocab"] * size, "flops": 4 * total * case["vocab"]}
    lengths, rows = _lengths(case)
    width = case["kv_heads"] * case["head"]
    if kind == "append":
        # rows in, codes out; the read-back's codes in and values out
        again = sum(l + r - l // case["page"] * case["page"] for l, r in zip(lengths, rows))
        return {"bytes": 2 * width * (sum(rows) * (size + 1) + again * 5), "flops": 4 * width * sum(rows)}
    q = case["heads"] * case["head"]
    cached = sum(l + r for l, r in zip(lengths, rows))
    pairs = sum(r * l + r * (r + 1) // 2 for l, r in zip(lengths, rows))
    return {"bytes": 2 * width * cached + sum(rows) * q * size * (3 if case["gate"] else 2), "flops": 4 * pairs * q}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    """The results from the definitions in 64 bits, one sequence and head at a time."""
    return globals()["_exact_" + case["kind"]](prepare(case, seed), case)


def _exact_rope(s, case):
    r, x = case["rotary"], s.x.double()
    if s.weight is not None:
        x = x / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + 1e-6) * s.weight.double()
    base, (factor, original, fast, slow, attention) = _rope_numbers(case)
    out = x.clone()
    for i in range(r // 2):
        theta = base ** (-2.0 * i / r)
        if case["scaling"] == "linear":
            theta /= factor
        elif case["scaling"] == "yarn":
            turns = lambda b: r * math.log(original / (b * 2 * math.pi)) / (2 * math.log(base))
            low, high = max(math.floor(turns(fast)), 0), min(math.ceil(turns(slow)), r - 1)
            ramp = min(1.0, max(0.0, (i - low) / max(high - low, 1e-3)))
            theta = theta * (1 - ramp) + theta / factor * ramp
        angle = s.positions.double() * theta
        c, w = attention * torch.cos(angle)[:, None], attention * torch.sin(angle)[:, None]
        j, k = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + r // 2)
        out[..., j], out[..., k] = x[..., j] * c - x[..., k] * w, x[..., j] * w + x[..., k] * c
    return out


def _exact_append(s, case):
    page, kv, head = case["page"], case["kv_heads"], case["head"]
    planes = [p[0].double() for p in _planes(s.storage, 1, s.pages, kv, page, head)]
    tables = s.tables.cpu().numpy()
    out, start = {"keys": [], "values": []}, 0
    for seq, (length, rows) in enumerate(zip(s.host_lengths, s.host_rows)):
        x = s.kv[start:start + rows].double()
        start += rows
        for name, plane, maxima, part in (("keys", planes[0], planes[2], 0), ("values", planes[1].transpose(2, 3), planes[3], 1)):
            for j in range(length // page, (length + rows - 1) // page + 1):
                begin, end = max(length, j * page), min(length + rows, (j + 1) * page)
                kept = begin - j * page
                v = x[begin - length:end - length, part].transpose(0, 1)     # [kv][tokens][head]
                top = v.abs().amax(dim=(1, 2))
                codes = plane[int(tables[seq, j])][:, :kept]
                if kept:
                    was = maxima[int(tables[seq, j])]
                    top = torch.maximum(top, was)
                    scaled = torch.round(codes * was[:, None, None] / top[:, None, None])
                    codes = torch.where((top > was)[:, None, None], scaled, codes)
                fresh = torch.round(v * 127.0 / top[:, None, None].clamp_min(1e-300))
                stored = torch.cat([codes, fresh], dim=1) * (top / 127.0)[:, None, None]
                out[name].append(stored.transpose(0, 1))
    return {name: torch.cat(parts) for name, parts in out.items()}


def _exact_attention(s, case):
    page, kv, head, heads = case["page"], case["kv_heads"], case["head"], case["heads"]
    keys, values, key_max, value_max = (p[0] for p in _planes(s.storage, 1, s.pages, kv, page, head))
    out = torch.empty(s.total, heads, head, dtype=torch.float64, device=DEV)
    start = 0
    for seq, (length, rows) in enumerate(zip(s.host_lengths, s.host_rows)):
        ids = s.tables[seq, :-(-(length + rows) // page)].long()
        mask = torch.arange(length + rows, device=DEV) <= length + torch.arange(rows, device=DEV)[:, None]
        for h in range(heads):
            g = h // (heads // kv)
            k = keys[ids, g].double() * key_max[ids, g].double()[:, None, None] / 127.0
            v = values[ids, g].double() * value_max[ids, g].double()[:, None, None] / 127.0
            k = k.reshape(-1, head)[:length + rows]
            v = v.transpose(1, 2).reshape(-1, head)[:length + rows]
            q = s.q[start:start + rows, h, 0].double()
            scores = (q @ k.t().contiguous()) * s.scale
            p = torch.softmax(scores.masked_fill(~mask, -math.inf), dim=-1)
            out[start:start + rows, h] = p @ v
        start += rows
    if case["gate"]:
        out = out * torch.sigmoid(s.q[:, :, 1].double())
    return out


def _exact_pages(s, case):
    return None  # bytes, not computed numbers


def _exact_verify(s, case):
    bounds = s.row_starts.tolist()
    logprobs = []
    tokens = s.tokens.tolist()
    uniforms = s.uniforms.double().tolist()
    for seq in range(case["sequences"]):
        first, end = bounds[seq], bounds[seq + 1]
        t = float(s.temperatures[seq])
        wait = None
        for row in range(first, end):
            if wait is not None:
                logprobs.append(0.0)
                continue
            logs = torch.log_softmax(s.target[row].double() / (t if t > 0 else 1.0), dim=0)
            p = torch.exp(logs)
            best = int(torch.nonzero(p == p.max())[0])
            if row + 1 < end:
                x = tokens[row + 1]
                if s.draft is None:
                    q = torch.zeros_like(p)
                    q[x] = 1.0
                else:
                    q = torch.softmax(s.draft[row].double() / (t if t > 0 else 1.0), dim=0)
                if (x == best) if t <= 0 else (uniforms[row] * float(q[x]) < float(p[x])):
                    logprobs.append(float(logs[x]))
                    continue
                left = torch.clamp(p - q, min=0.0)
                left = left if float(left.sum()) > 0 else p
            else:
                left = p
            if t <= 0:
                wait = best
            else:
                c = torch.cumsum(left, dim=0)
                found = torch.nonzero((c > uniforms[end - 1] * c[-1]) & (left > 0))
                wait = int(found[0]) if len(found) else int(torch.nonzero(left > 0)[-1])
            logprobs.append(float(logs[wait]))
    return {"logprobs": torch.tensor(logprobs, dtype=torch.float64, device=DEV), "accepted": None, "tokens": None}
