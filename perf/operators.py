"""The work of serving and training on packed sequences, as measurable cases.

Every case is one pass through one of these public calls:

    prompt   ``packed_attention`` over whole prompts of different lengths, packed along the tokens
    train    the same with its three gradients
    store    ``KeyValueCache.write`` (quantising), and with ``back`` ``KeyValueCache.read`` of the same rows
    draft    ``cached_attention`` of ``drafts`` new tokens a sequence over what the cache holds (1: a plain decode step)

``own`` chooses between the package's kernels and the operators written out in elementary torch operations, in float32.
Run with the repository's root as the working folder.
"""
import os
import random
import sys

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
BYTES = {"fp16": 2, "bf16": 2, "int8": 1, "e4m3": 1}
TOP = {"int8": 127.0, "e4m3": 448.0}          # largest value that a quantised row holds
CHUNK = 1 << 28                                # scores that the plain form holds at once
DEFAULTS = {"drafts": 0, "tree": False, "cache": "", "page": 0, "back": False}


def _package():
    path = os.path.abspath("experiments-pytorch-cuda-extension-for-sparse-matmul_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import sparse
    return sparse


# ---- cases -------------------------------------------------------------------------------------------
def _case(name, path, dtype, lengths, heads, groups, dim, **more):
    """``lengths``: tokens of every sequence (of the cache, for ``draft``; the first is the number of rows, for ``store``);
    ``heads``: key heads, ``groups``: query heads of each."""
    case = {"path": path, "dtype": dtype, "lengths": " ".join(str(n) for n in lengths), "heads": heads, "groups": groups,
            "dim": dim}
    case.update(DEFAULTS)
    case.update(more)
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
        # a batch of prompts of very different lengths for a model with grouped heads
        _case("prompt_bf16_grouped", "prompt", "bf16", [4096, 1531, 97, 2048, 421], 4, 4, 128),
        # one long document, eight query heads to a key head
        _case("prompt_fp16_long", "prompt", "fp16", [16384], 2, 8, 64),
        # a training step on short packed texts, every head with keys of its own
        _case("train_bf16_ragged", "train", "bf16", [512, 1000, 77, 1, 900, 1500], 12, 1, 64),
        # a training step on documents with grouped heads of 128
        _case("train_fp16_grouped", "train", "fp16", [4096, 2976, 1119], 4, 4, 128),
        # the new token of each of 48 sequences goes into the cache: latency
        _case("store_int8_step", "store", "bf16", [48], 4, 1, 128, cache="int8", page=64),
        # a prompt goes into the cache and is read back for the next stretch of it
        _case("store_e4m3_prompt", "store", "bf16", [8191], 8, 1, 128, cache="e4m3", page=32, back=True),
        # a batch of long prompts at once
        _case("store_int8_long", "store", "fp16", [65521], 8, 1, 64, cache="int8", page=128, back=True),
        # a decode step of 16 sequences, some of them just begun
        _case("decode_e4m3_batch", "draft", "bf16", [0, 1, 31, 32] + _spread(7, 12, 256, 8192), 4, 4, 128, drafts=1,
              cache="e4m3", page=64),
        # a decode step over one very long document
        _case("decode_int8_long", "draft", "fp16", [131071], 2, 8, 128, drafts=1, cache="int8", page=128),
        # a tree of 27 drafted tokens for each of four sequences, the cache in 16 bits
        _case("tree_bf16", "draft", "bf16", [8192, 4100, 2047, 700], 4, 4, 128, drafts=27, tree=True, cache="bf16", page=64),
        # the largest: 61 drafted tokens of each of 48 sequences
        _case("tree_int8_batch", "draft", "fp16", _spread(11, 48, 1024, 16384), 4, 4, 64, drafts=61, tree=True, cache="int8",
              page=32),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng: random.Random):
    path = rng.choice(["prompt", "prompt", "train", "train", "store", "draft", "draft", "draft"])
    dtype, dim, heads = rng.choice(["fp16", "bf16"]), rng.choice([64, 128]), rng.choice([1, 2, 3, 4, 8])
    groups = rng.choice([1, 2, 3, 4, 8])
    cache, page = rng.choice(["int8", "e4m3", dtype]), rng.choice([32, 64, 128, 256])
    if path == "store":
        kind = rng.choice(["int8", "e4m3"])
        return _case("", path, dtype, [_log_int(rng, 1, 65536)], heads, 1, dim, cache=kind, page=page,
                     back=kind == "e4m3" or rng.random() < 0.5)
    if path == "draft":
        count, drafts = _log_int(rng, 1, 48), rng.choice([1, 1, 2, _log_int(rng, 3, 64)])
        top = min(131072, max(64, (1 << 21) // (count * heads)))
        lengths = [rng.choice([0, 1]) if rng.random() < 0.05 else _log_int(rng, 16, top) for _ in range(count)]
        return _case("", path, dtype, lengths, heads, groups, dim, drafts=drafts, tree=drafts > 1 and rng.random() < 0.7,
                     cache=cache, page=page)
    count = _log_int(rng, 1, 16)
    top = ((1 << (32 if path == "prompt" else 29)) / (heads * groups * count * dim / 64)) ** 0.5
    lengths = [rng.choice([0, 1]) if rng.random() < 0.1 else _log_int(rng, 2, min(16384, int(top))) for _ in range(count)]
    return _case("", path, dtype, lengths if sum(lengths) else [1], heads, groups, dim)


def _lengths(case):
    return [int(n) for n in case["lengths"].split()]


# ---- inputs ------------------------------------------------------------------------------------------
def _normal(gen, dtype, *shape):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _rows(gen, dtype, tokens, heads, dim):
    """Keys and values as layers give them: every head with a size of its own, a few channels much larger, tokens that differ."""
    size = torch.exp(0.7 * torch.randn((1, heads, dim), generator=gen, device="cuda"))
    token = torch.exp(0.5 * torch.randn((tokens, heads, 1), generator=gen, device="cuda"))
    return (torch.randn((tokens, heads, dim), generator=gen, device="cuda") * size * token).to(dtype)


def _tree_mask(rng, count, drafts):
    """Which drafted token sees which: itself and its ancestors, parents drawn among the tokens before it."""
    mask = np.zeros((count, drafts, drafts), dtype=bool)
    for b in range(count):
        for i in range(drafts):
            parent = rng.randint(max(-1, i - 8), i - 1)
            if parent >= 0:
                mask[b, i] = mask[b, parent]
            mask[b, i, i] = True
    return torch.from_numpy(mask).cuda()


def _inputs(case, seed):
    """Everything that the calls read, the same whoever computes: a dict of tensors and of plain values."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, lengths = DTYPES[case["dtype"]], _lengths(case)
    heads, groups, dim = case["heads"], case["groups"], case["dim"]
    if case["path"] in ("prompt", "train"):
        tokens = sum(lengths)
        x = {"q": 2 * _normal(gen, dtype, tokens, heads * groups, dim), "k": _normal(gen, dtype, tokens, heads, dim),
             "v": _normal(gen, dtype, tokens, heads, dim),
             "offsets": torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], dtype=torch.int32, device="cuda")}
        if case["path"] == "train":
            x["dout"] = _normal(gen, dtype, tokens, heads * groups, dim)
        return x
    page, rng = case["page"], random.Random(seed)
    if case["path"] == "store":
        tokens = lengths[0]
        step = tokens <= 64           # one place in a page of each sequence; otherwise whole pages, in any order
        pages, places = (tokens if step else -(-tokens // page)) + 2, np.random.RandomState(seed % (1 << 32))
        order = places.permutation(pages)
        slots = (order[:, None] * page + (places.randint(0, page, (pages, 1)) if step else np.arange(page)[None, :])).reshape(-1)[:tokens].copy()
        kept = [i for i in range(tokens) if i % 16 != 5]
        slots[5::16] = -1             # rows that are not kept: drafts that were refused, the padding of a batch
        return {"k": _rows(gen, dtype, tokens, heads, dim), "v": _rows(gen, dtype, tokens, heads, dim), "pages": pages,
                "slots": torch.from_numpy(slots.astype(np.int32)).cuda(), "kept": torch.tensor(kept, device="cuda")}
    count, drafts = len(lengths), case["drafts"]
    per = [-(-n // page) for n in lengths]
    order = list(range(sum(per) + 1))
    rng.shuffle(order)
    width = max(1, max(per))
    table = np.full((count, width), -1, dtype=np.int32)
    for b in range(count):
        table[b, :per[b]] = [order.pop() for _ in range(per[b])]
    pages, shape = sum(per) + 1, (sum(per) + 1, heads, page)
    x = {"q": 2 * _normal(gen, dtype, count, drafts, heads * groups, dim), "k": _normal(gen, dtype, count, drafts, heads, dim),
         "v": _normal(gen, dtype, count, drafts, heads, dim), "pages": pages, "table": torch.from_numpy(table).cuda(),
         "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
         "tree": _tree_mask(rng, count, drafts) if case["tree"] else None}
    if case["cache"] in TOP:
        for name in ("keys", "values"):
            if case["cache"] == "int8":
                held = (40 * torch.randn(shape + (dim,), generator=gen, device="cuda")).clamp_(-127, 127).to(torch.int8)
            else:
                held = (140 * torch.randn(shape + (dim,), generator=gen, device="cuda")).clamp_(-448, 448).to(DTYPES["e4m3"])
            x[name] = held
            x[name[:-1] + "_scales"] = torch.exp(0.3 * torch.randn(shape, generator=gen, device="cuda")) / (TOP[case["cache"]] / 3.2)
    else:
        for name in ("keys", "values"):
            x[name] = _normal(gen, dtype, *shape, dim)
    return x


def _scale(case):
    return case["dim"] ** -0.5


def prepare(case, seed):
    x = _inputs(case, seed)
    state = {"case": case, "x": x, "seed": seed}
    if case["path"] == "train":
        for name in ("q", "k", "v"):
            x[name].requires_grad_(own)
    if case["path"] == "store":
        shape, dtype = (x["pages"], case["heads"], case["page"]), DTYPES[case["cache"]]
        if own:
            state["cache"] = cache = _package().KeyValueCache(*shape[:2], case["dim"], dtype=dtype, page=case["page"], device="cuda")
            held = (cache.keys, cache.values, cache.key_scales, cache.value_scales)
        else:
            held = [torch.empty(shape + (case["dim"],), dtype=dtype, device="cuda") for _ in range(2)]
            held += [torch.empty(shape, device="cuda") for _ in range(2)]
        for t in held:
            t.view(torch.uint8).zero_()
        state["held"] = tuple(held)
    if case["path"] == "draft" and own:
        state["cache"] = cache = _package().KeyValueCache(x["pages"], case["heads"], case["dim"], dtype=DTYPES[case["cache"]],
                                                          page=case["page"], device="cuda")
        for name in ("keys", "values", "key_scales", "value_scales"):
            if name in x:
                getattr(cache, name).copy_(x.pop(name))
    return state


# ---- the operators in elementary operations ----------------------------------------------------------
def _softmax_rows(scores, visible):
    """Softmax over the last axis of what is visible; a row that sees nothing is zero."""
    scores = scores.masked_fill(~visible, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = weights.sum(-1, keepdim=True)
    return weights / torch.where(total == 0, torch.ones_like(total), total)


def _by_head(x, heads):
    """``[n, heads * groups, d]`` -> ``[heads, groups, n, d]`` in float32."""
    n, all_heads, d = x.shape
    return x.reshape(n, heads, all_heads // heads, d).permute(1, 2, 0, 3).float()


def _by_token(x, dtype):
    heads, groups, n, d = x.shape
    return x.permute(2, 0, 1, 3).reshape(n, heads * groups, d).to(dtype)


def _plain_packed(case, x):
    q, k, v, dout = x["q"], x["k"], x["v"], x.get("dout")
    heads, scale, dtype = case["heads"], _scale(case), q.dtype
    out = torch.zeros_like(q)
    grads = [torch.zeros_like(t) for t in (q, k, v)] if dout is not None else []
    begin = 0
    for n in _lengths(case):
        if n == 0:
            continue
        at = slice(begin, begin + n)
        begin += n
        qs, ks, vs = _by_head(q[at], heads), _by_head(k[at], heads), _by_head(v[at], heads)
        gs = _by_head(dout[at], heads) if dout is not None else None
        dk, dv = torch.zeros_like(ks), torch.zeros_like(vs)
        o, dq = torch.empty_like(qs), torch.empty_like(qs)
        rows = max(1, min(n, CHUNK // (n * heads * case["groups"])))
        for r in range(0, n, rows):
            part = slice(r, min(n, r + rows))
            visible = torch.arange(n, device=q.device)[None, :] <= torch.arange(part.start, part.stop, device=q.device)[:, None]
            p = _softmax_rows(torch.matmul(qs[:, :, part] * scale, ks.transpose(-1, -2)), visible)
            o[:, :, part] = torch.matmul(p, vs)
            if gs is not None:
                g = gs[:, :, part]
                dv += torch.matmul(p.transpose(-1, -2), g).sum(1, keepdim=True)
                ds = p * (torch.matmul(g, vs.transpose(-1, -2)) - (g * o[:, :, part]).sum(-1, keepdim=True))
                dq[:, :, part] = torch.matmul(ds, ks) * scale
                dk += torch.matmul(ds.transpose(-1, -2), qs[:, :, part]).sum(1, keepdim=True) * scale
        out[at] = _by_token(o, dtype)
        if gs is not None:
            for total, one in zip(grads, (dq, dk, dv)):
                total[at] = _by_token(one, dtype)
    return (out, *grads) if grads else out


def _plain_quantise(x, kind):
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    held = x * TOP[kind] / torch.where(top == 0, torch.ones_like(top), top)
    held = held.round().to(torch.int8) if kind == "int8" else held.to(DTYPES["e4m3"])
    return held, (top / TOP[kind]).squeeze(-1)


def _plain_store(case, x, held):
    kind, page, kept = case["cache"], case["page"], x["kept"]
    slots = x["slots"][kept].long()
    at, place = slots // page, slots % page
    read = []
    for rows, values, scales in ((x["k"], held[0], held[2]), (x["v"], held[1], held[3])):
        q, s = _plain_quantise(rows[kept], kind)
        values.view(torch.uint8)[at, :, place] = q.view(torch.uint8)
        scales[at, :, place] = s
        if case["back"]:
            back = torch.zeros_like(rows)
            back[kept] = (values.view(torch.uint8)[at, :, place].view(values.dtype).float() * scales[at, :, place][..., None]).to(rows.dtype)
            read.append(back)
    return tuple(read) if read else held


def _plain_draft(case, x):
    heads, groups, page, dim = case["heads"], case["groups"], case["page"], case["dim"]
    q, table = x["q"], x["table"].long()
    count, drafts = q.shape[:2]
    width, span = table.size(1), max(1, CHUNK // (heads * groups * drafts * table.size(1) * page))
    outs = []
    for b in range(0, count, span):
        part = slice(b, b + span)
        n = table[part].size(0)
        pages = table[part].clamp(min=0)

        def gathered(name):
            held = x[name][pages] if case["cache"] != "e4m3" else x[name].view(torch.uint8)[pages].view(DTYPES["e4m3"])
            held = held.float()
            if case["cache"] in TOP:
                held = held * x[name[:-1] + "_scales"][pages][..., None]
            held = held.permute(0, 2, 1, 3, 4).reshape(n, heads, width * page, dim)
            new = x[name[0]][part].permute(0, 2, 1, 3).float()
            return torch.cat([held, new], 2)

        keys, values = gathered("keys"), gathered("values")
        qs = q[part].reshape(n, drafts, heads, groups, dim).permute(0, 2, 3, 1, 4).reshape(n, heads, groups * drafts, dim)
        scores = torch.matmul(qs.float() * _scale(case), keys.transpose(-1, -2))
        known = torch.arange(width * page, device=q.device)[None, :] < x["lengths"][part][:, None]
        tree = x["tree"][part] if x["tree"] is not None else torch.tril(torch.ones(n, drafts, drafts, dtype=torch.bool, device=q.device))
        visible = torch.cat([known[:, None, :].expand(n, drafts, width * page), tree], 2)
        visible = visible[:, None, None].expand(n, 1, groups, drafts, visible.size(-1)).reshape(n, 1, groups * drafts, -1)
        p = _softmax_rows(scores, visible)
        o = torch.matmul(p, values).reshape(n, heads, groups, drafts, dim).permute(0, 3, 1, 2, 4)
        outs.append(o.reshape(n, drafts, heads * groups, dim).to(q.dtype))
    return torch.cat(outs)


# ---- one pass ----------------------------------------------------------------------------------------
def run(state):
    case, x = state["case"], state["x"]
    if not own:
        with torch.no_grad():
            if case["path"] == "store":
                return _plain_store(case, x, state["held"])
            return _plain_draft(case, x) if case["path"] == "draft" else _plain_packed(case, x)
    sparse = _package()
    if case["path"] == "store":
        state["cache"].write(x["k"], x["v"], x["slots"])
        return state["cache"].read(x["slots"], x["k"].dtype) if case["back"] else state["held"]
    if case["path"] == "draft":
        return sparse.cached_attention(x["q"], x["k"], x["v"], state["cache"], x["table"], x["lengths"], tree=x["tree"],
                                       scale=_scale(case))
    out = sparse.packed_attention(x["q"], x["k"], x["v"], x["offsets"], scale=_scale(case), causal=True)
    if case["path"] == "prompt":
        return out
    return (out,) + torch.autograd.grad(out, (x["q"], x["k"], x["v"]), x["dout"])


def work(case):
    """Bytes and operations of one pass: every operand read once, every result written once."""
    lengths, heads, groups, dim, es = _lengths(case), case["heads"], case["groups"], case["dim"], BYTES[case["dtype"]]
    if case["path"] in ("prompt", "train"):
        tokens, pairs = sum(lengths), sum(n * (n + 1) // 2 for n in lengths)
        items, product = 2 * tokens * heads * (groups + 1) * dim, 2.0 * heads * groups * dim * pairs
        train = case["path"] == "train"       # as many items again in gradients; five more products
        return {"bytes": es * items * (2 if train else 1), "flops": product * (7 if train else 2)}
    if case["path"] == "store":
        kept = sum(1 for i in range(lengths[0]) if i % 16 != 5)
        row, held = es * heads * dim, heads * (BYTES[case["cache"]] * dim + 4)
        moved = kept * (row + held) + (kept * held + lengths[0] * row if case["back"] else 0)
        return {"bytes": 2 * moved + 4 * lengths[0] * (2 if case["back"] else 1), "flops": 6.0 * kept * heads * dim}
    drafts, count = case["drafts"], len(lengths)
    held = BYTES[case["cache"]] * dim + (4 if case["cache"] in TOP else 0)
    return {"bytes": 2 * sum(lengths) * heads * held + 2 * es * count * drafts * heads * (groups + 1) * dim,
            "flops": 4.0 * heads * groups * dim * drafts * (sum(lengths) + count * (drafts + 1) / 2)}


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------
def _exact_attention(q, k, v, scale, visible):
    """Rows ``q [n, d]`` over ``k``, ``v [m, d]``, all float64: weights and result."""
    s = torch.where(visible, scale * (q @ k.t()), torch.full((), -np.inf, dtype=torch.float64, device=q.device))
    if not s.size(1):
        return s, torch.zeros_like(q)
    e = torch.exp(s - torch.nan_to_num(s.max(dim=1, keepdim=True).values, neginf=0.0))
    e[~visible] = 0.0
    total = e.sum(dim=1, keepdim=True)
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    return p, p @ v


def _exact_e4m3(x):
    """Nearest multiple of the step at each value: eight steps to a power of two, 2^-9 below 2^-6; ties to even."""
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    step = torch.exp2(exponent - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    x, scale = _inputs(case, seed), _scale(case)
    heads, groups, dim, lengths = case["heads"], case["groups"], case["dim"], _lengths(case)
    if case["path"] in ("prompt", "train"):
        pairs = heads * groups * sum(n * n for n in lengths) * dim / 64
        if pairs > 6e9:
            return None
        train = case["path"] == "train"
        results = [torch.zeros(x[name].shape, dtype=torch.float64, device="cuda") for name in (("q", "q", "k", "v") if train else "q")]
        for b, n in enumerate(lengths):
            first = sum(lengths[:b])
            for h in range(heads * groups):
                g = h // groups
                for r in range(0, n, 4096):
                    mine, seen = slice(first + r, first + min(n, r + 4096)), slice(first, first + min(n, r + 4096))
                    q, k, v = x["q"][mine, h].double(), x["k"][seen, g].double(), x["v"][seen, g].double()
                    causal = torch.ones(q.size(0), k.size(0), dtype=torch.bool, device="cuda").tril(r)
                    p, o = _exact_attention(q, k, v, scale, causal)
                    results[0][mine, h] = o
                    if train:
                        d = x["dout"][mine, h].double()
                        ds = scale * p * (d @ v.t() - (d * o).sum(1, keepdim=True))
                        results[1][mine, h] = ds @ k
                        results[2][seen, g] += ds.t() @ q
                        results[3][seen, g] += p.t() @ d
        return tuple(results) if train else results[0]
    if case["path"] == "store":
        kind, page = case["cache"], case["page"]
        shape = (x["pages"], heads, page)
        held, scales, back = [], [], []
        slots = x["slots"].cpu().numpy()
        kept = np.nonzero(slots >= 0)[0]
        for name in ("k", "v"):
            rows = x[name].double()
            top = rows.abs().max(dim=-1, keepdim=True).values
            y = torch.where(top > 0, rows * TOP[kind] / top, torch.zeros_like(rows))
            y = torch.round(y) if kind == "int8" else _exact_e4m3(y)
            s = top / TOP[kind]
            read = torch.zeros_like(rows)
            read[kept] = (y * s)[kept]
            back.append(read)
            whole, factors = torch.zeros(shape + (dim,), dtype=torch.float64, device="cuda"), torch.zeros(shape, dtype=torch.float64, device="cuda")
            where = torch.from_numpy(slots[kept].astype(np.int64)).cuda()
            whole[where // page, :, where % page] = y[kept]
            factors[where // page, :, where % page] = s[kept, :, 0]
            held.append(whole.to(torch.int8) if kind == "int8" else whole)
            scales.append(factors)
        return tuple(back) if case["back"] else (*held, *scales)
    drafts, page, count = case["drafts"], case["page"], len(lengths)
    if heads * groups * drafts * sum(lengths) * dim > 2e11 or count * heads * groups > 4000:
        return None
    result = torch.zeros(x["q"].shape, dtype=torch.float64, device="cuda")
    table = x["table"].cpu().numpy()
    for b, n in enumerate(lengths):
        used = torch.from_numpy(table[b, :-(-n // page)].astype(np.int64)).cuda()
        for g in range(heads):
            both = []
            for name in ("keys", "values"):
                rows = x[name].view(torch.uint8)[used, g].view(x[name].dtype).double()
                if case["cache"] in TOP:
                    rows = rows * x[name[:-1] + "_scales"][used, g].double()[..., None]
                both.append(torch.cat([rows.reshape(-1, dim)[:n], x[name[0]][b, :, g].double()]))
            seen = torch.ones(drafts, n + drafts, dtype=torch.bool, device="cuda")
            seen[:, n:] = x["tree"][b] if x["tree"] is not None else torch.ones(drafts, drafts, dtype=torch.bool, device="cuda").tril()
            for h in range(g * groups, (g + 1) * groups):
                result[b, :, h] = _exact_attention(x["q"][b, :, h].double(), *both, scale, seen)[1]
    return result
