"""What sequences keep from one call to the next, as measurable cases: recurrent states and pages of a cache.

Every case is one pass through these public calls:

    prompt    ``packed_linear_attention`` over packed prompts of different lengths, with ``states`` from given states to the final ones
    train     the same with its gradients
    step      ``linear_attention_step``: one token of every sequence, states updated in place
    grow      ``PageTable.append`` for new tokens, and ``KeyValueCache.write`` of their keys and values
    fork      ``PageTable.fork``: every parent continued by several children, and ``KeyValueCache.copy`` of the pages that this takes
    compact   ``PageTable.compact`` of a table in long use, and ``KeyValueCache.copy`` of the pages that move

``own`` chooses between the package's kernels and the operators written out in elementary torch operations, in float32.
Run with the repository's root as the working folder.
"""
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8}
BYTES = {"fp16": 2, "bf16": 2, "int8": 1}
CHUNK = 128                                    # tokens of a chunk of the plain form
DEFAULTS = {"states": False, "copies": 0, "cache": "", "page": 0, "held": "", "spare": 0}


def _package():
    path = os.path.abspath("experiments-pytorch-cuda-extension-for-sparse-matmul_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import sparse
    return sparse


# ---- cases -------------------------------------------------------------------------------------------
def _case(name, path, dtype, lengths, heads, groups, dim, **more):
    """``lengths``: tokens of every sequence (``step``: how many sequences; ``grow``: new tokens; ``fork``: of every parent);
    ``heads``: key heads, ``groups``: query heads of each; ``held``: tokens that sequences have before they ``grow``; ``spare``: pages
    nobody has; ``copies``: children of every parent."""
    case = {"path": path, "dtype": dtype, "lengths": " ".join(str(n) for n in lengths), "heads": heads, "groups": groups,
            "dim": dim}
    case.update(DEFAULTS)
    case.update(more)
    case["held"] = " ".join(str(n) for n in case["held"]) if case["held"] else ""
    if name:
        case["name"] = name
    return case


def _spread(seed, count, low, high):
    """``count`` lengths between ``low`` and ``high``, evenly over their logarithm."""
    rng = random.Random(seed)
    return [_log_int(rng, low, high) for _ in range(count)]


def listed():
    return [
        # a few short prompts that arrive together, one of a single token, one empty: latency
        _case("prompt_fp16_short", "prompt", "fp16", [1, 37, 0, 200, 130], 12, 1, 64),
        # the next stretches of documents of very different lengths, grouped heads, states kept for the steps that follow
        _case("prompt_bf16_long", "prompt", "bf16", [40000, 9001, 97, 16000, 421], 4, 2, 128, states=True),
        # a training step on short packed texts
        _case("train_bf16_ragged", "train", "bf16", [512, 1000, 77, 1, 900, 1500], 12, 1, 64),
        # the largest: a training step on long documents whose states come from the part before
        _case("train_fp16_long", "train", "fp16", [16384, 8191], 16, 1, 128, states=True),
        # the next token of a few sequences: latency
        _case("step_fp16_few", "step", "fp16", [3], 4, 1, 64),
        # the next token of a full batch, grouped heads
        _case("step_bf16_batch", "step", "bf16", [250], 16, 2, 128),
        # a decode step: the sequences of a batch grow by one token, some are idle
        _case("grow_int8_step", "grow", "bf16", [1, 1, 0, 1] * 16, 4, 1, 128, cache="int8", page=64, held=_spread(5, 64, 16, 4096),
              spare=200),
        # prompts arrive while others are being answered
        _case("grow_bf16_prompts", "grow", "bf16", [0] * 24 + _spread(6, 24, 64, 4096), 8, 1, 128, cache="bf16", page=32,
              held=_spread(7, 24, 64, 8192) + [0] * 24, spare=1500),
        # four continuations of each of three prompts
        _case("fork_fp16_few", "fork", "fp16", [700, 129, 64], 4, 1, 64, copies=4, cache="fp16", page=32, spare=20),
        # sixty-three continuations of each of eight prompts, most of them long
        _case("fork_int8_many", "fork", "bf16", [16383, 9000, 4097, 12345, 800, 30000, 6001, 65], 8, 1, 128, copies=63, cache="int8",
              page=128, spare=600),
        # a small cache with a few holes
        _case("compact_int8_few", "compact", "bf16", _spread(9, 7, 30, 1000), 4, 1, 64, cache="int8", page=32, spare=12),
        # a cache in long use of which half is free again: what is left moves together
        _case("compact_bf16_half", "compact", "bf16", _spread(8, 48, 512, 16384), 4, 1, 128, cache="bf16", page=64, spare=3200),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng: random.Random):
    path = rng.choice(["prompt", "prompt", "train", "train", "step", "grow", "fork", "compact"])
    dtype, dim, heads = rng.choice(["fp16", "bf16"]), rng.choice([64, 128]), rng.choice([1, 2, 3, 4, 8, 12])
    groups = rng.choice([1, 1, 2, 3, 4])
    if path == "step":
        return _case("", path, dtype, [_log_int(rng, 1, (250 * 16 * 2 * 128 * 128) // (heads * groups * dim * dim))], heads, groups, dim)
    if path in ("prompt", "train"):
        count = _log_int(rng, 1, 16)
        top = (1 << (26 if path == "prompt" else 24)) // (heads * groups * count * dim)
        lengths = [rng.choice([0, 1]) if rng.random() < 0.1 else _log_int(rng, 2, max(3, min(65536, top))) for _ in range(count)]
        return _case("", path, dtype, lengths if sum(lengths) else [1], heads, groups, dim, states=rng.random() < 0.5)
    cache, page, count = rng.choice(["int8", dtype]), rng.choice([32, 64, 128, 256]), _log_int(rng, 1, 48)
    top = max(64, (1 << 17) // count)
    lengths = [_log_int(rng, 1, min(16384, top)) for _ in range(count)]
    spare = _log_int(rng, 16, 1024)
    if path == "grow":
        new = [rng.choice([0, 1]) for _ in lengths] if rng.random() < 0.5 else [rng.choice([0, _log_int(rng, 1, min(4096, top))]) for _ in lengths]
        new[rng.randrange(count)] = 1
        spare += sum(-(-n // page) + 1 for n in new)
        return _case("", path, dtype, new, heads, 1, dim, cache=cache, page=page, held=lengths, spare=spare)
    if path == "fork":
        copies = _log_int(rng, 1, max(2, 384 // count))
        return _case("", path, dtype, lengths, heads, 1, dim, cache=cache, page=page, copies=copies, spare=spare + count * copies)
    return _case("", path, dtype, lengths, heads, 1, dim, cache=cache, page=page, spare=spare)


def _numbers(text):
    return [int(n) for n in text.split()]


# ---- inputs ------------------------------------------------------------------------------------------
def _normal(gen, dtype, *shape):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _log_decay(gen, heads):
    """Memories from one token and a half to a thousand tokens."""
    return -torch.exp2(-0.5 - 9.5 * torch.rand((heads,), generator=gen, device="cuda"))


def _int32(values):
    return torch.from_numpy(np.asarray(values, dtype=np.int32)).cuda()


def _offsets(lengths):
    return _int32(np.concatenate([[0], np.cumsum(lengths, dtype=np.int64)]))


def _pages_in_use(case, seed):
    """A table in long use: every sequence's pages anywhere in the cache.  Lengths of the sequences, table, uses (numpy)."""
    rng, page, lengths = np.random.RandomState(seed % (1 << 32)), case["page"], _numbers(case["lengths"])
    room = list(lengths)                            # tokens that a row has to have room for
    if case["path"] == "grow":
        room = [a + b for a, b in zip(_numbers(case["held"]), lengths)]
        lengths = _numbers(case["held"])
    elif case["path"] == "fork":                    # children hold what is left of other answers
        room = lengths + [lengths[i // case["copies"]] for i in range(len(lengths) * case["copies"])]
        room += [2 * page]
        lengths = lengths + [int(n) for n in rng.randint(0, 2 * page, len(lengths) * case["copies"])]
    per = [-(-n // page) for n in lengths]
    pages = case["spare"] + sum(-(-n // page) for n in _numbers(case["held"] or case["lengths"]))
    if case["path"] == "fork":
        pages += 2 * (len(lengths) - len(_numbers(case["lengths"])))
    order = rng.permutation(pages)
    table = np.full((len(lengths), max(1, max(-(-n // page) for n in room))), -1, dtype=np.int32)
    uses, at = np.zeros(pages, dtype=np.int32), 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    uses[order[:at]] = 1
    return np.asarray(lengths, dtype=np.int32), table, uses


def _inputs(case, seed):
    """Everything that the calls read, the same whoever computes: a dict of tensors and of plain values."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, lengths = DTYPES[case["dtype"]], _numbers(case["lengths"])
    heads, groups, dim = case["heads"], case["groups"], case["dim"]
    if case["path"] in ("prompt", "train", "step"):
        tokens = sum(lengths)
        x = {"q": _normal(gen, dtype, tokens, heads * groups, dim), "k": _normal(gen, dtype, tokens, heads, dim),
             "v": _normal(gen, dtype, tokens, heads, dim), "log_decay": _log_decay(gen, heads)}
        if case["path"] == "step":
            slots = np.random.RandomState(seed % (1 << 32)).permutation(tokens + 3)[:tokens]
            if tokens > 8:
                slots[5] = -1                       # a row of the batch that is idle
            x["slots"] = _int32(slots)
            x["states"] = 4 * torch.randn((tokens + 3, heads, dim, dim), generator=gen, device="cuda")
            return x
        x["offsets"] = _offsets(lengths)
        if case["states"]:
            x["states"] = 4 * torch.randn((len(lengths), heads, dim, dim), generator=gen, device="cuda")
        if case["path"] == "train":
            x["dout"] = _normal(gen, dtype, tokens, heads * groups, dim)
            if case["states"]:
                x["dlast"] = torch.randn((len(lengths), heads, dim, dim), generator=gen, device="cuda")
        return x
    held, table, uses = _pages_in_use(case, seed)
    x = {"lengths": _int32(held), "table": _int32(table), "uses": _int32(uses)}
    shape = (len(uses), heads, case["page"], dim)
    if case["path"] == "grow":
        x["k"], x["v"] = _normal(gen, dtype, sum(lengths), heads, dim), _normal(gen, dtype, sum(lengths), heads, dim)
        x["offsets"] = _offsets(lengths)
    if case["path"] == "fork":
        count, copies = len(lengths), case["copies"]
        x["parents"] = _int32(np.repeat(np.arange(count), copies))
        x["children"] = _int32(count + np.arange(count * copies))
    for name in ("keys", "values"):
        if case["cache"] == "int8":
            x[name] = torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)
            x[name[:-1] + "_scales"] = torch.exp(0.3 * torch.randn(shape[:3], generator=gen, device="cuda")) / 40
        else:
            x[name] = _normal(gen, DTYPES[case["cache"]], *shape)
    return x


def _scale(case):
    return case["dim"] ** -0.5


HELD = ("keys", "values", "key_scales", "value_scales")
TABLE = ("table", "lengths", "uses")


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": case, "x": x}
    if case["path"] == "train":
        for name in ("q", "k", "v", "states"):
            if name in x:
                x[name].requires_grad_(own)
    if case["cache"]:
        state["first"] = [x[name].clone() for name in TABLE]
        if own:
            sparse = _package()
            cache = sparse.KeyValueCache(x["keys"].size(0), case["heads"], case["dim"], dtype=DTYPES[case["cache"]], page=case["page"])
            for name in HELD:
                if name in x:
                    getattr(cache, name).copy_(x.pop(name))
            table = sparse.PageTable(cache.pages, case["page"], x["table"].size(0), x["table"].size(1))
            for name in TABLE:
                getattr(table, name).copy_(x.pop(name))
            state["cache"], state["pages"] = cache, table
        state["now"] = [getattr(state["pages"], name) if own else x[name] for name in TABLE]
        state["held"] = [t for t in ((getattr(state["cache"], name) if own else x.get(name)) for name in HELD) if t is not None]
    return state


# ---- linear attention in elementary operations ---------------------------------------------------------
def _powers(log_decay, exponents):
    """decay ** exponents, [heads, ...]; zero where the exponent is negative; in 64 bits, the products take 32."""
    e = torch.as_tensor(exponents, dtype=torch.float64, device=log_decay.device)
    p = torch.exp(log_decay.double().reshape(-1, *([1] * e.dim())) * e.clamp(min=0))
    return torch.where(e >= 0, p, torch.zeros_like(p)).float()


class _Chunks:
    """Packed tokens as chunks of CHUNK, each of one sequence; ``turned``: every sequence from its end."""

    def __init__(self, lengths, log_decay, turned):
        c, first, place, index, chunk_of, ordinal = CHUNK, 0, [], [], [], []
        for b, n in enumerate(lengths):
            i = np.arange(n, dtype=np.int64)
            at = c * len(chunk_of) + i
            place.append(at)
            index.append(first + (n - 1 - i if turned else i))
            chunk_of += [b] * -(-n // c)
            ordinal += list(range(-(-n // c)))
            first += n
        self.place, self.index = (torch.from_numpy(np.concatenate(t)).cuda() for t in (place, index))
        self.count, owner, ordinal = len(chunk_of), np.asarray(chunk_of, dtype=np.int64), np.asarray(ordinal, dtype=np.int64)
        n = np.asarray(lengths, dtype=np.int64)
        t = np.arange(c)
        inside = np.minimum(c, n[owner] - c * ordinal)                          # tokens of a chunk
        same = owner[:, None] == owner[None, :]
        # from the end of chunk i to the beginning of chunk j, both of one sequence
        gap = np.where(same & (ordinal[:, None] > ordinal[None, :]), c * (ordinal[:, None] - ordinal[None, :] - 1), -1)
        left = np.where(np.arange(len(n))[:, None] == owner[None, :], n[None, :][0][:, None] - np.minimum(c * (ordinal + 1), n[owner])[None, :], -1)
        self.within = _powers(log_decay, t[:, None] - t[None, :])               # [heads, c, c]
        self.since = _powers(log_decay, t + 1)                                  # from a chunk's beginning to after its token t
        self.until = _powers(log_decay, inside[:, None] - 1 - t[None, :])       # [heads, chunks, c]: from a token to its chunk's end
        self.between = _powers(log_decay, gap)                                  # [heads, chunks, chunks]
        self.start = _powers(log_decay, c * ordinal)                            # [heads, chunks]: from the sequence's start
        self.last = _powers(log_decay, left)                                    # [heads, sequences, chunks]: from a chunk's end to the last token
        self.whole = _powers(log_decay, n)                                      # [heads, sequences]
        self.owner = torch.from_numpy(owner).cuda()

    def split(self, x):
        """``[tokens, heads, d]`` -> ``[heads, chunks, CHUNK, d]`` in float32."""
        flat = torch.zeros((self.count * CHUNK,) + x.shape[1:], dtype=torch.float32, device=x.device)
        flat[self.place] = x.float()[self.index]
        return flat.reshape(self.count, CHUNK, x.size(1), x.size(2)).permute(2, 0, 1, 3)

    def join(self, x, tokens):
        """The way back: ``[tokens, heads, d]`` in float32."""
        out = torch.zeros((tokens, x.size(0), x.size(3)), dtype=torch.float32, device=x.device)
        out[self.index] = x.permute(1, 2, 0, 3).reshape(-1, x.size(0), x.size(3))[self.place]
        return out

    def walk(self, a, b, c, first):
        """sum over s <= t of decay^(t - s) (a_t . b_s) c_s, plus decay^(t + 1) a_t times ``first [heads, sequences, d, d]``; and the
        decayed sum of b_s c_s^T after the last token."""
        out = torch.matmul(torch.matmul(a, b.transpose(-1, -2)) * self.within[:, None], c)
        heads, d = b.size(0), b.size(3)
        sums = torch.matmul((b * self.until[..., None]).transpose(-1, -2), c)                 # [heads, chunks, d, d]
        flat = sums.reshape(heads, self.count, d * d)
        states = torch.matmul(self.between, flat).reshape(sums.shape)
        last = torch.matmul(self.last, flat).reshape(heads, -1, d, d)
        if first is not None:
            states = states + self.start[..., None, None] * first[:, self.owner]
            last = last + self.whole[..., None, None] * first
        # a state is followed by the decay of the token that meets it
        return out + torch.matmul(a * self.since[:, None, :, None], states), last


def _plain_linear(case, x):
    groups, scale, dtype, lengths = case["groups"], _scale(case), x["q"].dtype, _numbers(case["lengths"])
    tokens, many = sum(lengths), lambda t: None if t is None else t.repeat_interleave(groups, 0)
    decay = x["log_decay"].repeat_interleave(groups)
    first = x["states"].transpose(0, 1) if "states" in x else None              # [heads, sequences, d, d]
    along = _Chunks(lengths, decay, False)
    q, k, v = along.split(x["q"]), many(along.split(x["k"])), many(along.split(x["v"]))
    out, last = along.walk(q, k, v, many(first))
    outs = [(scale * along.join(out, tokens)).to(dtype)]
    if first is not None:
        outs.append(last[::groups].transpose(0, 1).contiguous())
    if case["path"] == "prompt":
        return tuple(outs)
    summed = lambda t: t.reshape(t.size(0), -1, groups, t.size(2)).sum(2)       # over the query heads of a key head
    dout = along.split(x["dout"])
    dq, _ = along.walk(dout, v, k, many(first).transpose(-1, -2) if first is not None else None)
    back = _Chunks(lengths, decay, True)
    q, k, v, dout = back.split(x["q"]), many(back.split(x["k"])), many(back.split(x["v"])), back.split(x["dout"])
    # backwards the state in front of a token has no decay of its own: what comes from the end is one decay less
    end = x["dlast"].transpose(0, 1) / scale if first is not None else None
    share = None
    if end is not None:
        share = torch.zeros_like(end).repeat_interleave(groups, 0)
        share[::groups] = end / torch.exp(x["log_decay"].double()).float()[:, None, None, None]
    dv, start = back.walk(k, q, dout, share)
    dk, _ = back.walk(v, dout, q, share.transpose(-1, -2) if share is not None else None)
    outs += [(scale * along.join(dq, tokens)).to(dtype)]
    outs += [(scale * summed(back.join(t, tokens))).to(dtype) for t in (dk, dv)]
    if first is not None:
        start = start.reshape(-1, groups, *start.shape[1:]).sum(1) * torch.exp(x["log_decay"].double()).float()[:, None, None, None]
        outs.append((scale * start).transpose(0, 1).contiguous())
    return tuple(outs)


def _plain_step(case, x):
    groups, states, slots = case["groups"], x["states"], x["slots"].long()
    kept = slots >= 0
    at = slots[kept]
    k, v = x["k"][kept].float(), x["v"][kept].float()
    now = torch.exp(x["log_decay"].double()).float()[:, None, None] * states[at] + k[..., :, None] * v[..., None, :]
    states[at] = now
    q = x["q"][kept].float().reshape(k.size(0), k.size(1), groups, -1)
    out = torch.zeros_like(x["q"])
    out[kept] = (_scale(case) * torch.matmul(q, now)).reshape(k.size(0), -1, k.size(2)).to(out.dtype)
    return out, states


# ---- pages in elementary operations --------------------------------------------------------------------
def _lowest_free(uses, count):
    return torch.nonzero(uses == 0)[:count, 0]


def _plain_grow(case, x):
    table, lengths, uses = (x[name] for name in TABLE)
    page, offsets = case["page"], x["offsets"].long()
    new, held = offsets.diff(), lengths.long()
    had, has = (held + page - 1) // page, (held + new + page - 1) // page
    need = has - had
    ends = need.cumsum(0)
    fits = (ends <= (uses == 0).sum()) & (has <= table.size(1))                 # all of these do
    taken = _lowest_free(uses, int(ends[-1]))
    column = torch.arange(table.size(1), device=table.device)[None, :]
    fresh = (column >= had[:, None]) & (column < has[:, None]) & fits[:, None]
    table[fresh] = taken.int()
    uses[taken] = 1
    owner = torch.searchsorted(offsets, torch.arange(x["k"].size(0), device=table.device), right=True) - 1
    place = held[owner] + torch.arange(x["k"].size(0), device=table.device) - offsets[owner]
    at, place = table[owner, place // page].long(), place % page
    lengths += torch.where(fits, new, torch.zeros_like(new)).int()
    for rows, name in ((x["k"], "keys"), (x["v"], "values")):
        if case["cache"] == "int8":
            top = rows.float().abs().amax(-1, keepdim=True)
            x[name][at, :, place] = (rows.float() * 127 / torch.where(top == 0, torch.ones_like(top), top)).round().to(torch.int8)
            x[name[:-1] + "_scales"][at, :, place] = (top / 127).squeeze(-1)
        else:
            x[name][at, :, place] = rows
    return (at * page + place).int()


def _plain_copy(x, sources, targets):
    kept = sources >= 0
    for name in HELD:
        if name in x:
            x[name].view(torch.uint8)[targets[kept].long()] = x[name].view(torch.uint8)[sources[kept].long()]


def _plain_fork(case, x):
    table, lengths, uses = (x[name] for name in TABLE)
    page, parents, children = case["page"], x["parents"].long(), x["children"].long()
    column = torch.arange(table.size(1), device=table.device)[None, :]
    rows, new = table[parents], lengths[parents].long()
    own_pages = column < ((lengths[children].long() + page - 1) // page)[:, None]
    left = table[children][own_pages].long()
    uses.index_add_(0, left, torch.full_like(left, -1, dtype=torch.int32))
    shared = column < (new // page)[:, None]
    also = rows[shared].long()
    uses.index_add_(0, also, torch.ones_like(also, dtype=torch.int32))
    partial = new % page > 0                        # no parent is a child here: every child needs such a page of its own
    targets, sources = torch.full_like(x["parents"], -1), torch.full_like(x["parents"], -1)
    taken = _lowest_free(uses, int(partial.sum()))
    targets[partial] = taken.int()
    sources[partial] = rows[partial, new[partial] // page]
    uses[taken] = 1
    rows = torch.where(shared, rows, torch.full_like(rows, -1))
    rows[partial, new[partial] // page] = taken.int()
    table[children] = rows
    lengths[children] = new.int()
    _plain_copy(x, sources, targets)
    return sources, targets


def _plain_compact(case, x):
    table, lengths, uses = (x[name] for name in TABLE)
    count = int((uses > 0).sum())
    holes = torch.nonzero(uses[:count] == 0)[:, 0]
    moved = torch.nonzero(uses[count:] > 0)[:, 0] + count
    sources, targets = torch.full((uses.numel() // 2,), -1, dtype=torch.int32, device=uses.device), torch.full((uses.numel() // 2,), -1, dtype=torch.int32, device=uses.device)
    sources[:moved.numel()] = moved.int()
    targets[:moved.numel()] = holes.int()
    number = torch.arange(uses.numel() + 1, dtype=torch.int32, device=uses.device)
    number[moved] = holes.int()
    number[-1] = -1                                 # of the table's empty places
    table.copy_(number[table.long()])
    uses[holes] = uses[moved]
    uses[moved] = 0
    _plain_copy(x, sources, targets)
    return sources, targets


# ---- one pass ----------------------------------------------------------------------------------------
def run(state):
    case, x = state["case"], state["x"]
    if case["cache"]:
        if case["path"] != "fork":                  # the same batch over again; a fork leaves its own parents as they are
            for now, first in zip(state["now"], state["first"]):
                now.copy_(first)
        if not own:
            made = {"grow": _plain_grow, "fork": _plain_fork, "compact": _plain_compact}[case["path"]](case, x)
        elif case["path"] == "grow":
            made = state["pages"].append(x["offsets"], x["k"].size(0))
            state["cache"].write(x["k"], x["v"], made)
        else:
            made = state["pages"].fork(x["parents"], x["children"]) if case["path"] == "fork" else state["pages"].compact()
            state["cache"].copy(*made)
        return (*(made if isinstance(made, tuple) else (made,)), *state["now"], *state["held"])
    if not own:
        with torch.no_grad():
            return _plain_step(case, x) if case["path"] == "step" else _plain_linear(case, x)
    sparse = _package()
    if case["path"] == "step":
        return sparse.linear_attention_step(x["q"], x["k"], x["v"], x["log_decay"], x["states"], x["slots"], scale=_scale(case)), x["states"]
    out = sparse.packed_linear_attention(x["q"], x["k"], x["v"], x["log_decay"], x["offsets"], scale=_scale(case), states=x.get("states"),
                                         return_states=case["states"])
    outs = out if case["states"] else (out,)
    if case["path"] == "prompt":
        return outs
    leaves = [x[name] for name in ("q", "k", "v", "states") if name in x]
    return outs + torch.autograd.grad(outs, leaves, [x["dout"], x["dlast"]] if case["states"] else [x["dout"]])


def work(case):
    """Bytes and operations of one pass: every operand read once, every result written once."""
    lengths, heads, groups, dim, es = _numbers(case["lengths"]), case["heads"], case["groups"], case["dim"], BYTES[case["dtype"]]
    if case["path"] in ("prompt", "train", "step"):
        tokens, state = sum(lengths), 4 * heads * dim * dim
        rows = 2 * tokens * heads * (groups + 1) * dim * es                     # q, k, v, the result
        update, use = 2.0 * tokens * heads * dim * dim, 2.0 * tokens * heads * groups * dim * dim
        if case["path"] == "step":
            return {"bytes": rows + 2 * tokens * state, "flops": update + use}
        held = 2 * len(lengths) * state if case["states"] else 0
        if case["path"] == "prompt":
            return {"bytes": rows + held, "flops": update + use}
        # gradients: as many rows and states again; dq, dk, dv from their states, and the other state's products
        return {"bytes": 2 * rows + 2 * held, "flops": update + 2 * use + 3 * use}
    page, item = case["page"], BYTES[case["cache"]] * dim + (4 if case["cache"] == "int8" else 0)
    one = 2 * heads * page * item                                               # a page of the cache
    if case["path"] == "grow":
        tokens = sum(lengths)
        return {"bytes": tokens * heads * 2 * (es * dim + item) + 8 * tokens, "flops": 2.0 * tokens * heads * dim}
    if case["path"] == "fork":
        entries = sum(-(-n // page) for n in lengths) * case["copies"]
        return {"bytes": 2 * one * case["copies"] * sum(1 for n in lengths if n % page) + 8 * entries, "flops": float(entries)}
    used = sum(-(-n // page) for n in lengths)
    pages = used + case["spare"]
    return {"bytes": 2 * one * round(used * (1 - used / pages)) + 4 * (pages + used), "flops": float(pages)}


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------
def _exact_linear(case, x):
    """Token by token: S_t = decay S_(t-1) + k_t v_t^T, o_t = scale q_t S_t; sequences side by side, the longest first."""
    lengths, heads, groups, dim, scale = _numbers(case["lengths"]), case["heads"], case["groups"], case["dim"], _scale(case)
    order = sorted(range(len(lengths)), key=lambda b: -lengths[b])
    begin = torch.tensor([sum(lengths[:b]) for b in order], device="cuda")
    decay = torch.exp(x["log_decay"].double())[None, :, None, None]
    alive = [sum(1 for b in order if lengths[b] > t) for t in range(lengths[order[0]])]
    grouped = lambda t: t.double().reshape(t.size(0), heads, groups, dim)
    k, v, q = x["k"].double(), x["v"].double(), grouped(x["q"])
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    s = torch.zeros((len(lengths), heads, dim, dim), dtype=torch.float64, device="cuda")
    if "states" in x:
        s.copy_(x["states"].double()[order])
    g = grouped(x["dout"]) if case["path"] == "train" else None
    for t, n in enumerate(alive):
        at = begin[:n] + t
        s[:n] = decay * s[:n] + k[at][..., :, None] * v[at][..., None, :]
        out[at] = scale * torch.matmul(q[at], s[:n])
        if g is not None:
            dq[at] = scale * torch.matmul(g[at], s[:n].transpose(-1, -2).contiguous())
    back = [order.index(b) for b in range(len(lengths))]
    outs = [out.reshape(x["q"].shape)] + ([s[back]] if "states" in x else [])
    if g is None:
        return tuple(outs)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    r = torch.zeros_like(s)                         # the gradient of S_t
    last = x["dlast"].double()[order] if "states" in x else None
    if last is not None:
        r.copy_(last)
    for t in range(len(alive) - 1, -1, -1):
        n = alive[t]
        at = begin[:n] + t
        r[:n] += scale * torch.matmul(q[at].transpose(-1, -2).contiguous(), g[at])
        dk[at] = torch.matmul(r[:n], v[at][..., None])[..., 0]
        dv[at] = torch.matmul(k[at][..., None, :], r[:n])[..., 0, :]
        r[:n] = decay * r[:n]
    return tuple(outs + [dq.reshape(x["q"].shape), dk, dv] + ([r[back]] if "states" in x else []))


def _exact_pages(case, x):
    """The table's new state and what moves, one sequence after the other."""
    page, held, pages = case["page"], x["lengths"].cpu().numpy().copy(), x["uses"].numel()
    width = x["table"].size(1)
    rows = [list(row[:-(-int(n) // page)]) for row, n in zip(x["table"].cpu().numpy(), held)]
    users = [0] * pages
    for row in rows:
        for p in row:
            users[p] += 1
    lowest = lambda: users.index(0)
    if case["path"] == "grow":
        slots = []
        for b, n in enumerate(_numbers(case["lengths"])):
            for _ in range(n):
                if held[b] % page == 0:
                    rows[b].append(lowest())
                    users[rows[b][-1]] = 1
                slots.append(rows[b][-1] * page + held[b] % page)
                held[b] += 1
        made = (slots,)
    elif case["path"] == "fork":
        parents, children = x["parents"].tolist(), x["children"].tolist()
        for c in children:
            for p in rows[c]:
                users[p] -= 1
        for a, c in zip(parents, children):
            held[c], rows[c] = held[a], list(rows[a])
            for p in rows[c][:held[a] // page]:
                users[p] += 1
        made = ([], [])
        for a, c in zip(parents, children):
            copied = held[a] % page > 0
            made[0].append(rows[a][-1] if copied else -1)
            made[1].append(lowest() if copied else -1)
            if copied:
                rows[c][-1] = made[1][-1]
                users[made[1][-1]] = 1
    else:
        count = sum(1 for n in users if n)
        sources = [p for p in range(count, pages) if users[p]]
        targets = [p for p in range(count) if not users[p]]
        to = dict(zip(sources, targets))
        rows = [[to.get(p, p) for p in row] for row in rows]
        for a, b in to.items():
            users[b], users[a] = users[a], 0
        nothing = [-1] * (pages // 2 - len(sources))
        made = (sources + nothing, targets + nothing)
    table = [list(row) + [-1] * (width - len(row)) for row in rows]
    return [_int32(t) for t in made], [_int32(table), _int32(held), _int32(users)]


def exact(case, seed):
    x = _inputs(case, seed)
    if case["path"] in ("prompt", "train"):
        return _exact_linear(case, x)
    if case["path"] == "step":
        kept, groups = x["slots"] >= 0, case["groups"]
        states, out = x["states"].double(), torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
        for h in range(case["heads"]):
            at = x["slots"][kept].long()
            now = torch.exp(x["log_decay"][h].double()) * states[at, h] + x["k"][kept, h].double()[:, :, None] * x["v"][kept, h].double()[:, None, :]
            states[at, h] = now
            for i in range(h * groups, (h + 1) * groups):
                out[kept, i] = _scale(case) * torch.matmul(x["q"][kept, i].double()[:, None, :], now)[:, 0]
        return out, states
    made, table = _exact_pages(case, x)
    if case["path"] == "grow":
        where = made[0].long()
        for name in ("keys", "values"):
            rows = x[name[0]].double()
            if case["cache"] == "int8":
                top = rows.abs().max(dim=-1, keepdim=True).values
                held, factors = torch.round(torch.where(top > 0, rows * 127 / top, torch.zeros_like(rows))).to(torch.int8), top[..., 0] / 127
                x[name[:-1] + "_scales"] = x[name[:-1] + "_scales"].double()
                x[name[:-1] + "_scales"][where // case["page"], :, where % case["page"]] = factors
            else:
                x[name], held = x[name].double(), rows
            x[name][where // case["page"], :, where % case["page"]] = held
    else:
        moves = [(a, b) for a, b in zip(made[0].tolist(), made[1].tolist()) if a >= 0]
        for name in HELD:
            if name in x and moves:
                x[name][[b for _, b in moves]] = x[name][[a for a, _ in moves]]
    return (*made, *table, *(x[name] for name in HELD if name in x))
