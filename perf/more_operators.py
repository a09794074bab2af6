"""Performance cases of sequences that share pages of the paged 4-bit KV cache:
several answers to one prompt, searches that branch, chats behind one long
instruction, drafts of which a part is kept.

Kinds (`kind` of a case):
  fork    ops.bind_paged_fork: sequences continued by any number of children,
          which share the whole pages and get the last one copied;
  free    ops.bind_paged_free: the pages that no sequence holds;
  move    ops.bind_paged_move: chosen keys and values put side by side in other
          pages, as they are in 4 bits;
  shared  ops.bind_paged_gqa_shared: causal attention of groups of sequences
          that have their first pages in common.

A pool is bytes [pages, kv_heads, page / 32, 40 * dim]: one block of 32 keys
of one KV head is 40 * dim bytes, laid out as _block_bytes() says.

Heads are the repository's (16 query / 4 KV heads of 256) and the 64 and 128
wide ones of its tests.
"""
import math

import torch

own = False


def listed():
    return [
        # sixteen answers to one prompt
        fork("fork_samples_16", 1, 16, 8191, 4, 256, 128),
        # a step of a search with many beams at many lengths, in large pages
        fork("fork_beams_64", 48, 64, 16381, 4, 256, 256),
        # a small server's tables
        free("free_16", 16, 256, 64, 4096),
        # a large one's, whose chats share many of their pages
        free("free_500", 500, 1031, 64, 400_000),
        # the rows of each chat's drafts that were right, out of the drafts' pages
        move("move_accept_16", 16, 5, 24, 8191, 4, 256, 64),
        # a quarter of a long context is kept
        move("move_evict_8k", 1, 8192, 32749, 4, 4, 256, 64),
        # histories of many lengths made shorter, to odd places of their pages
        move("move_ragged", 13, 901, 2003, 77, 8, 128, 32),
        # a few answers to a prompt of medium length: the smallest attention
        shared("shared_samples_8", 1, 8, 1, 4099, 200, 16, 4, 256, 64),
        # many chats behind one long instruction
        shared("shared_chats_48", 1, 48, 1, 16384, 1024, 16, 4, 256, 64),
        # drafts of a few tokens for answers about a long document
        shared("shared_drafts_16", 1, 16, 5, 32749, 500, 16, 4, 256, 128),
        # several instructions with chats of many lengths, eight query heads a KV head
        shared("shared_ragged", 6, 21, 2, 9001, 2001, 32, 4, 128, 32),
        # many short answers to two prompts, narrow heads
        shared("shared_narrow", 2, 100, 1, 7001, 300, 32, 8, 64, 256),
    ]


def _named(name, case):
    return case if name is None else {"name": name, **case}


def fork(name, parents, children, past, kv_heads, dim, page):
    return _named(name, {"kind": "fork", "parents": parents, "children": children, "past": past,
                         "kv_heads": kv_heads, "dim": dim, "page": page})


def free(name, sequences, width, page, pages):
    return _named(name, {"kind": "free", "sequences": sequences, "width": width, "page": page,
                         "pages": pages})


def move(name, sequences, rows, span, past, kv_heads, dim, page):
    """`rows` of `span` positions go behind `past`."""
    return _named(name, {"kind": "move", "sequences": sequences, "rows": rows, "span": span,
                         "past": past, "kv_heads": kv_heads, "dim": dim, "page": page})


def shared(name, groups, members, rows, prefix, rest, q_heads, kv_heads, dim, page):
    """`members` sequences a group, with `rows` rows each behind a prefix and up
    to `rest` keys of their own."""
    return _named(name, {"kind": "shared", "groups": groups, "members": members, "rows": rows,
                         "prefix": prefix, "rest": rest, "q_heads": q_heads, "kv_heads": kv_heads,
                         "dim": dim, "page": page})


def _log(rng, low, high):
    """A whole number from low to high, spread evenly over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choices(["fork", "free", "move", "shared"], [15, 15, 20, 50])[0]
    page = rng.choice([32, 64, 128, 256])
    if kind == "free":
        sequences, width = _log(rng, 1, 500), _log(rng, 1, 1031)
        return free(None, sequences, width, page, _log(rng, max(2, width // 3), 400_000))
    dim, kv_heads = rng.choice([256, 256, 128, 64]), rng.choice([1, 2, 4, 8])
    if kind == "fork":
        most = 64 * 4 * 256 * 256 // (kv_heads * dim * page)
        children = _log(rng, 1, min(256, most))
        return fork(None, _log(rng, 1, children), children, _log(rng, 1, 16384) - 1, kv_heads, dim, page)
    if kind == "move":
        sequences = _log(rng, 1, 32)
        rows = _log(rng, 1, 8192 * 4 * 256 // (sequences * kv_heads * dim))
        span = min(65536, rows * rng.choice([1, 2, 4, 4, 8]) + rng.randint(0, 9))
        return move(None, sequences, rows, max(rows, span), _log(rng, 1, 8192) - 1, kv_heads, dim, page)
    per = rng.choice([1, 2, 4, 4, 5, 8, 16])
    while per * kv_heads > 32:
        per = (per + 1) // 2
    groups, members = _log(rng, 1, 6), _log(rng, 1, 100)
    rows = 1 if rng.random() < 0.6 else rng.randint(2, 8)
    # the products of all pairs at most the 48 listed chats'
    pairs = 48 * 16384 * 4096 // (groups * members * rows * per * kv_heads * dim)
    prefix = _log(rng, page, max(page, min(32768, pairs)))
    rest = _log(rng, 1, max(1, min(2048, pairs // 8)))
    return shared(None, groups, members, rows, prefix, rest, per * kv_heads, kv_heads, dim, page)


# ---------------------------------------------------------------- lengths

def _part(n, i, least=0):
    """n for the first, between an eighth of it and all for the others."""
    return n if i == 0 else max(least, n * (2 + (i * 37 + 5) % 15) // 16)


def _parents(case):
    """The parent of every child: each has one, the other children have any."""
    n = case["parents"]
    return [i if i < n else (i * 37 + 5) % n for i in range(case["children"])]


def _groups(case):
    """(shared keys, [(rows, past) of each sequence]) of every group: whole
    pages are shared, what is left of the prefix is each sequence's own."""
    out, n = [], 0
    for g in range(case["groups"]):
        prefix, members = _part(case["prefix"], g, 1), _part(case["members"], g, 1)
        seqs = []
        for _ in range(members):
            seqs.append((_part(case["rows"], n, 1), prefix + _part(case["rest"], n)))
            n += 1
        out.append((prefix // case["page"] * case["page"], seqs))
    return out


# ----------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rows16(g, *shape):
    """Activations: normal, with a few channels of every head that are larger."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    large = 1 + 4 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.03).float()
    return (x * large).half()


def _pool(g, case, pages):
    """A pool whose blocks hold 32 keys and values each."""
    dim = case["dim"]
    pool = torch.empty(pages, case["kv_heads"], case["page"] // 32, 40 * dim, dtype=torch.uint8,
                       device="cuda")
    flat = pool.view(-1, 40 * dim)
    for at in range(0, flat.shape[0], 4096):
        part = flat[at:at + 4096]
        k, v = (_quantized(_rows16(g, part.shape[0], 32, dim)) for _ in range(2))
        part.copy_(_block_bytes(*k, *v))
    return pool


def _tables(g, counts, width, extra=3):
    """Rows of `width` page numbers, of which the first counts[s] are pages of a
    pool with `extra` more, in any order: (table, numbers of the others)."""
    order = torch.randperm(sum(counts) + extra, generator=g, device="cuda").int()
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    return table, order[at:]


def prepare(case, seed):
    g = _gen(seed)
    state = {"case": case}
    return {"fork": _prepare_fork, "free": _prepare_free, "move": _prepare_move,
            "shared": _prepare_shared}[case["kind"]](case, state, g)


def _prepare_fork(case, state, g):
    parents, children, page = case["parents"], case["children"], case["page"]
    past = [_part(case["past"], s) for s in range(parents)]
    counts = [-(-p // page) for p in past]
    width = max(counts) + 2
    table, spare = _tables(g, counts, width, children + 3)
    return state | {"pool": _pool(g, case, sum(counts) + children + 3), "table": table,
                    "past": _ints(past), "parent": _ints(_parents(case)),
                    "spare": spare[:children].contiguous(),
                    "table_out": torch.zeros(children, width, dtype=torch.int32, device="cuda"),
                    "past_out": torch.zeros(children, dtype=torch.int32, device="cuda")}


def _prepare_free(case, state, g):
    sequences, width, pages = case["sequences"], case["width"], case["pages"]
    lengths = [_part(width * case["page"], s) for s in range(sequences)]
    # half of a row's pages are those of one prompt, the others its own
    table = torch.randint(pages, (sequences, width), generator=g, device="cuda").int()
    table[:, :width // 2] = table[0, :width // 2]
    return state | {"table": table, "lengths": _ints(lengths),
                    "free": torch.zeros(pages, dtype=torch.int32, device="cuda"),
                    "count": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _prepare_move(case, state, g):
    sequences, page = case["sequences"], case["page"]
    rows = [_part(case["rows"], s, 1) for s in range(sequences)]
    span = [max(r, _part(case["span"], s)) for s, r in enumerate(rows)]
    past = [_part(case["past"], s) for s in range(sequences)]
    counts = [-(-n // page) for n in span] + [-(-(p + r) // page) for p, r in zip(past, rows)]
    both, _ = _tables(g, counts, max(counts))
    chosen = [torch.randperm(n, generator=g, device="cuda")[:r].sort()[0] for n, r in zip(span, rows)]
    return state | {"pool": _pool(g, case, sum(counts) + 3),
                    "source_table": both[:sequences].contiguous(),
                    "table": both[sequences:].contiguous(), "past": _ints(past),
                    "starts": _ints([0] + rows).cumsum(0).int(), "source": torch.cat(chosen).int()}


def _prepare_shared(case, state, g):
    page, groups = case["page"], _groups(case)
    seqs = [s for _, members in groups for s in members]
    rows, past = [r for r, _ in seqs], [p for _, p in seqs]
    # a group's shared pages, then each sequence's own
    common = [keys // page for keys, _ in groups]
    owned = [-(-(r + p) // page) - n for n, (_, members) in zip(common, groups) for r, p in members]
    parts, _ = _tables(g, common + owned, max(1, max(common), max(owned)))
    table = torch.full((len(seqs), max(-(-(r + p) // page) for r, p in seqs)), -1, dtype=torch.int32,
                       device="cuda")
    s = 0
    for n, (_, members) in enumerate(groups):
        for _ in members:
            table[s, :common[n]] = parts[n, :common[n]]
            table[s, common[n]:common[n] + owned[s]] = parts[len(groups) + s, :owned[s]]
            s += 1
    q = _rows16(g, sum(rows), case["q_heads"], case["dim"])
    return state | {"pool": _pool(g, case, sum(common) + sum(owned) + 3), "table": table,
                    "past": _ints(past), "starts": _ints([0] + rows).cumsum(0).int(),
                    "groups": _ints([0] + [len(m) for _, m in groups]).cumsum(0).int(),
                    "prefix": _ints([keys for keys, _ in groups]), "q": q, "out": torch.empty_like(q)}


# ------------------------------------------------------- the 4-bit format

def _quantized(x):
    """(codes, scale, bias) of groups of 32 channels: x fp16 [..., dim]."""
    x = x.float().unflatten(-1, (-1, 32))
    low, high = x.amin(-1), x.amax(-1)
    scale = ((high - low) / 15.0).half()
    s = scale.float()
    bias = (low - 16.0 * s).half()
    steps = (x - bias.float()[..., None]) / torch.where(s > 0, s, torch.inf)[..., None]
    return (torch.round(steps) - 16.0).clamp(0, 15).to(torch.uint8), scale, bias


def _values(codes, scale, bias):
    """fp16((16 + code) * scale + bias), the value a code stands for."""
    x = (16.0 + codes.double()) * scale.double()[..., None] + bias.double()[..., None]
    return x.half().flatten(-2)


# Key 16 m + 8 t + 4 h + v of a block is row 8 m + 4 h + v of its tile t for
# keys, and nibble slot 4 t + v of word 2 m + h for values. Slot e (and, for
# keys, channel e of a word's eight) is nibble e / 2 + 4 (e % 2).
_NIBBLE = [0, 4, 1, 5, 2, 6, 3, 7]
_SLOT_OF_NIBBLE = [0, 2, 4, 6, 1, 3, 5, 7]


def _packed(slots):
    """Bytes [..., 4] of the eight nibbles in slots [..., 8]."""
    nibbles = slots[..., _SLOT_OF_NIBBLE]
    return nibbles[..., 0::2] | nibbles[..., 1::2] << 4


def _spread(data):
    """The eight slots of words given as bytes [..., 4]."""
    return torch.stack((data & 15, data >> 4), -1).flatten(-2)[..., _NIBBLE]


def _block_bytes(kc, ks, kb, vc, vs, vb):
    """Blocks [n, 40 dim] of the keys' and values' codes [n, 32, groups, 32]
    and scales and biases [n, 32, groups]."""
    n, _, groups, _ = kc.shape
    dim, lane = 32 * groups, 32 if groups >= 4 else 16
    keys = (2, 2, 2, 4)  # m, t, h, v
    # keys: [t][channels / (4 lane)][quarter][m h v][word][byte]
    k = kc.reshape(n, *keys, dim // (4 * lane), 4, lane // 8, 8).permute(0, 2, 5, 6, 1, 3, 4, 7, 8)
    k = _packed(k).reshape(n, -1)
    # their scale and bias: [t][group][m h v][2]
    km = torch.stack((ks, kb), -1).view(n, *keys, groups, 2).permute(0, 2, 5, 1, 3, 4, 6)
    km = km.reshape(n, -1).view(torch.uint8)
    # values: [channel / 64][m h][channel % 16][channel / 16 % 4][byte], slots t v
    v = vc.reshape(n, *keys, dim // 64, 4, 16).permute(0, 5, 1, 3, 7, 6, 2, 4).flatten(-2)
    v = _packed(v).reshape(n, -1)
    # their scales, then biases: [group][2][m h t v]
    vm = torch.stack((vs, vb), -1).view(n, *keys, groups, 2).permute(0, 5, 6, 1, 3, 2, 4)
    vm = vm.reshape(n, -1).view(torch.uint8)
    return torch.cat((k, km, v, vm), 1)


def _block_parts(data):
    """The arguments of _block_bytes() that give these blocks."""
    n, dim = data.shape[0], data.shape[1] // 40
    lane, groups = 32 if dim >= 128 else 16, dim // 32
    k, km, v, vm = data.split((16 * dim, 4 * dim, 16 * dim, 4 * dim), 1)
    k = _spread(k.reshape(n, 2, dim // (4 * lane), 4, 2, 2, 4, lane // 8, 4))
    k = k.permute(0, 4, 1, 5, 6, 2, 3, 7, 8).reshape(n, 32, groups, 32)
    km = km.contiguous().view(torch.float16).view(n, 2, groups, 2, 2, 4, 2)
    km = km.permute(0, 3, 1, 4, 5, 2, 6).reshape(n, 32, groups, 2)
    v = _spread(v.reshape(n, dim // 64, 2, 2, 16, 4, 4)).unflatten(-1, (2, 4))
    v = v.permute(0, 2, 6, 3, 7, 1, 5, 4).reshape(n, 32, groups, 32)
    vm = vm.contiguous().view(torch.float16).view(n, groups, 2, 2, 2, 2, 4)
    vm = vm.permute(0, 3, 5, 4, 6, 1, 2).reshape(n, 32, groups, 2)
    return [x.clone() for x in (k, km[..., 0], km[..., 1], v, vm[..., 0], vm[..., 1])]


# ------------------------------------------------------------- plain forms

def run(state):
    if own:
        return _run_own(state)
    return {"fork": _plain_fork, "free": _plain_free, "move": _plain_move,
            "shared": _plain_shared}[state["case"]["kind"]](state)


def _plain_fork(state):
    pool, page = state["pool"], state["case"]["page"]
    parent = state["parent"].long()
    past = state["past"][parent]
    width = state["table"].shape[1]
    slot, last = torch.arange(width, device="cuda"), (past // page)[:, None]
    table = state["table"][parent]
    table = torch.where(slot < last, table, torch.where(slot == last, state["spare"][:, None], -1))
    # the blocks of the last page that hold keys
    child, block = torch.nonzero(torch.arange(page // 32, device="cuda") * 32 < (past % page)[:, None],
                                 as_tuple=True)
    source = state["table"][parent[child], past[child].long() // page].long()
    pool[state["spare"][child].long(), :, block] = pool[source, :, block]
    return {"pool": pool, "table": table, "past": past}


def _plain_free(state):
    pages, page = state["case"]["pages"], state["case"]["page"]
    slot = torch.arange(state["table"].shape[1], device="cuda")
    held = torch.zeros(pages, dtype=torch.bool, device="cuda")
    held[state["table"][slot * page < state["lengths"][:, None]].long()] = True
    numbers = torch.arange(pages, device="cuda", dtype=torch.int32)
    order = torch.sort(held.to(torch.uint8), stable=True)[1]  # the free ones first
    free = torch.where(held[order], -1, numbers[order])
    return {"free": free, "count": (~held).sum(0, keepdim=True).int()}


def _places(state, positions, seq, table):
    """(page, block of it, key of that) of positions of sequences."""
    page = state["case"]["page"]
    return state[table][seq, positions // page].long(), positions % page // 32, positions % 32


def _plain_move(state):
    pool = state["pool"]
    heads, dim = state["case"]["kv_heads"], state["case"]["dim"]
    row = torch.arange(state["source"].numel(), device="cuda")
    seq = torch.searchsorted(state["starts"][1:], row, right=True)

    def blocks_of(page, block):
        where, at = torch.unique(page * pool.shape[2] + block, return_inverse=True)
        where = (where // pool.shape[2], slice(None), where % pool.shape[2])
        return where, at, _block_parts(pool[where].flatten(0, 1))

    page, block, key = _places(state, state["source"].long(), seq, "source_table")
    _, at, parts = blocks_of(page, block)
    moved = [p.view(-1, heads, *p.shape[1:])[at, :, key] for p in parts]
    to = state["past"][seq].long() + row - state["starts"][seq]
    page, block, key = _places(state, to, seq, "table")
    where, at, parts = blocks_of(page, block)
    for part, rows in zip(parts, moved):
        part.view(-1, heads, *part.shape[1:])[at, :, key] = rows
    pool[where] = _block_bytes(*parts).view(-1, heads, 40 * dim)
    return {"pool": pool}


def _plain_cached(state, pages):
    """K and V fp32 [..., kv_heads, keys, dim] of pages [..., n]."""
    heads, dim = state["case"]["kv_heads"], state["case"]["dim"]
    blocks = state["pool"][pages.clamp(min=0).long()].movedim(-3, -4)  # [..., kv_heads, n, blocks, bytes]
    keys = pages.shape[-1] * state["case"]["page"]
    parts = _block_parts(blocks.reshape(-1, 40 * dim))
    return [_values(*p).float().view(*pages.shape[:-1], heads, keys, dim) for p in (parts[:3], parts[3:])]


def _plain_shared(state):
    case = state["case"]
    page, dim, heads = case["page"], case["dim"], case["kv_heads"]
    per = case["q_heads"] // heads
    out = torch.empty(state["q"].shape, dtype=torch.float32, device="cuda")
    s = at = 0
    for keys, members in _groups(case):
        n, most = len(members), max(r for r, _ in members)
        total = sum(r for r, _ in members)
        rest = max(r + p for r, p in members) - keys
        seqs = slice(s, s + n)
        # the rows of every sequence, padded to the longest
        row = torch.arange(total, device="cuda") + at
        seq = torch.searchsorted(state["starts"][s + 1:s + n + 1], row, right=True)
        i = row - state["starts"][seqs][seq]
        q = torch.zeros(n, heads, most, per, dim, device="cuda")
        q[seq, :, i] = state["q"][at:at + total].view(-1, heads, per, dim).float()
        # scores of the shared keys, then of the sequence's own
        k, v = _plain_cached(state, state["table"][s, :keys // page])
        k_own, v_own = _plain_cached(state, state["table"][seqs, keys // page:-(-(keys + rest) // page)])
        common = q.transpose(0, 1).reshape(heads, n * most * per, dim) @ k.transpose(-1, -2).contiguous()
        scores = q.flatten(2, 3) @ k_own.transpose(-1, -2).contiguous()
        position = keys + torch.arange(scores.shape[-1], device="cuda")
        last = state["past"][seqs, None] + torch.arange(most, device="cuda")
        hidden = position > last.repeat_interleave(per, 1)[..., None]
        scores.masked_fill_(hidden[:, None], -torch.inf)
        common = common.view(heads, n, most * per, keys).transpose(0, 1)
        weights = torch.cat((common, scores), -1) / math.sqrt(dim)
        weights = (weights - weights.amax(-1, keepdim=True)).exp()
        sums = weights.sum(-1, keepdim=True)
        common, scores = weights.split((keys, scores.shape[-1]), -1)
        both = common.transpose(0, 1).reshape(heads, n * most * per, keys) @ v
        both = both.view(heads, n, most * per, dim).transpose(0, 1) + scores @ v_own
        rows = (both / sums).view(n, heads, most, per, dim)[seq, :, i]
        out[at:at + total] = rows.reshape(total, -1, dim)
        s, at = s + n, at + total
    return out.half()


# ------------------------------------------------------- the framework's

def _run_own(state):
    from llminfer_amd import ops

    kind = state["case"]["kind"]
    if "call" not in state:  # bound once, as a serving loop keeps it
        if kind == "fork":
            state["call"] = ops.bind_paged_fork(state["pool"], state["table"], state["past"],
                                                state["parent"], state["spare"], state["table_out"],
                                                state["past_out"])
        elif kind == "free":
            state["call"] = ops.bind_paged_free(state["table"], state["lengths"], state["case"]["page"],
                                                state["free"], state["count"])
        elif kind == "move":
            state["call"] = ops.bind_paged_move(state["pool"], state["starts"], state["past"],
                                                state["table"], state["source"], state["source_table"])
        else:
            state["call"] = ops.bind_paged_gqa_shared(state["q"], state["pool"], state["starts"],
                                                      state["past"], state["table"], state["groups"],
                                                      state["prefix"], state["out"])
    state["call"]()
    if kind == "fork":
        return {"pool": state["pool"], "table": state["table_out"], "past": state["past_out"]}
    if kind == "free":
        return {"free": state["free"], "count": state["count"]}
    return {"pool": state["pool"]} if kind == "move" else state["out"]


# ------------------------------------------------------------------- work

def work(case):
    if case["kind"] == "free":
        held = sum(-(-_part(case["width"] * case["page"], s) // case["page"])
                   for s in range(case["sequences"]))
        return {"bytes": 4 * (held + case["pages"] + case["sequences"] + 1), "flops": 0}
    row = case["kv_heads"] * case["dim"] * 1.25  # a key and its value, in bytes
    if case["kind"] == "fork":
        # the blocks with keys of the parents' last pages, one copy a child, and the tables
        past = [_part(case["past"], s) for s in range(case["parents"])]
        last = [-(-(p % case["page"]) // 32) * 32 for p in past]
        most, parents = max(past) // case["page"] + 3, _parents(case)
        return {"bytes": (sum(last[p] for p in parents) + sum(last[p] for p in set(parents))) * row
                + 4 * (sum(past) // case["page"] + len(parents) * most), "flops": 0}
    if case["kind"] == "move":
        rows = sum(_part(case["rows"], s, 1) for s in range(case["sequences"]))
        return {"bytes": rows * (2 * row + 4), "flops": 0}
    groups = _groups(case)
    seqs = [(keys, r, p) for keys, members in groups for r, p in members]
    keys = sum(k for k, _ in groups) + sum(r + p - k for k, r, p in seqs)
    pairs = sum(r * p + r * (r + 1) // 2 for _, r, p in seqs)
    heads = case["q_heads"] * case["dim"]
    return {"bytes": keys * row + sum(r for _, r, _ in seqs) * heads * 4, "flops": 4 * heads * pairs}


# ------------------------------------------------- the definitions, 64 bits

def _key64(data, dim):
    """Where a block keeps a key's channels: [32, dim] of (byte, shift) of the
    code and byte of the scale, and the same of the value; biases are 2 and 64
    bytes behind the scale."""
    key = torch.arange(32, device=data.device)[:, None]
    channel = torch.arange(dim, device=data.device)[None]
    m, t, h, v = key >> 4, key >> 3 & 1, key >> 2 & 1, key & 3
    per = 32 if dim >= 128 else 16
    nib = channel % 8 // 2 + channel % 2 * 4
    lane = channel // per % 4 * 16 + 8 * m + 4 * h + v
    k_at = t * 8 * dim + channel // (4 * per) * 32 * per + lane * (per // 2) + channel % per // 8 * 4
    k_scale = 16 * dim + t * 2 * dim + (channel // 32 * 16 + 8 * m + 4 * h + v) * 4
    slot = 4 * t + v
    v_nib = slot // 2 + slot % 2 * 4
    v_at = 20 * dim + channel // 64 * 1024 + ((2 * m + h) * 16 + channel % 16) * 16 + channel // 16 % 4 * 4
    v_scale = 36 * dim + channel // 32 * 128 + ((2 * m + h) * 8 + slot) * 2
    return ((k_at + nib // 2, (nib % 2 * 4).expand(32, dim), k_scale, 2),
            (v_at + v_nib // 2, (v_nib % 2 * 4).expand(32, dim), v_scale, 64))


def _cached64(state, pages, head):
    """K and V [keys, dim] of pages, one KV head, by the definition."""
    dim = state["case"]["dim"]
    data = state["pool"][pages.long(), head].view(-1, 40 * dim)
    halves, out = data.view(torch.float16).double(), []
    for at, shift, scale, bias in _key64(data, dim):
        code = (data[:, at] >> shift.to(torch.uint8)) & 15
        x = (16 + code.double()) * halves[:, scale // 2] + halves[:, (scale + bias) // 2]
        out.append(x.half().double().view(-1, dim))
    return out


def _moved64(state):
    """The pool's bytes behind a move: code by code and scale by scale."""
    dim, page, pool = state["case"]["dim"], state["case"]["page"], state["pool"].clone()
    data, starts = pool.view(-1, 40 * dim), state["starts"].tolist()
    per_page = page // 32
    heads = torch.arange(pool.shape[1], device="cuda")
    places = _key64(data, dim)

    def blocks(pages, positions):  # of every head: [heads, rows]
        return ((pages.long() * pool.shape[1])[None] + heads[:, None]) * per_page + positions % page // 32

    rows = []
    for s, (a, b) in enumerate(zip(starts, starts[1:])):
        source = state["source"][a:b].long()
        target = state["past"][s].long() + torch.arange(b - a, device="cuda")
        rows.append((blocks(state["source_table"][s][source // page], source), source % 32,
                     blocks(state["table"][s][target // page], target), target % 32))
    source, key, target, to = (torch.cat(x, -1) for x in zip(*rows))
    old = data.clone()
    for at, shift, scale, bias in places:
        code = (old[source[..., None], at[key]] >> shift[key].to(torch.uint8)) & 15
        for nibble in (0, 4):  # two channels or keys share a byte: one of them at a time
            row, channel = (shift[to] == nibble).nonzero(as_tuple=True)
            index = target[:, row], at[to[row], channel].expand(target.shape[0], -1)
            data[index] = data[index] & (240 >> nibble) | code[:, row, channel] << nibble
        for half in (0, 1, bias, bias + 1):
            data[target[..., None], scale[to] + half] = old[source[..., None], scale[key] + half]
    return pool


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "free":
        lengths, table = state["lengths"].tolist(), state["table"].cpu()
        held = set()
        for s, n in enumerate(lengths):
            held.update(table[s, :-(-n // case["page"])].tolist())
        free = [p for p in range(case["pages"]) if p not in held]
        return {"free": _ints(free + [-1] * len(held)), "count": _ints([len(free)])}
    if case["kind"] == "move":
        return {"pool": _moved64(state)}
    page = case["page"]
    if case["kind"] == "fork":
        pool, past, width = state["pool"], state["past"].tolist(), state["table"].shape[1]
        table, spare = state["table"].tolist(), state["spare"].tolist()
        rows, lengths = [], []
        for i, p in enumerate(state["parent"].tolist()):
            whole, rest = divmod(past[p], page)
            rows.append(table[p][:whole] + [spare[i]] + [-1] * (width - whole - 1))
            lengths.append(past[p])
            if rest:
                blocks = (rest + 31) // 32
                pool[spare[i], :, :blocks] = pool[table[p][whole], :, :blocks]
        return {"pool": pool, "table": _ints(rows), "past": _ints(lengths)}
    per = case["q_heads"] // case["kv_heads"]
    out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    s = at = 0
    for keys, members in _groups(case):
        for head in range(case["kv_heads"]):
            k0, v0 = _cached64(state, state["table"][s, :keys // page], head)
            row = at
            for i, (r, p) in enumerate(members):
                k1, v1 = _cached64(state, state["table"][s + i, keys // page:-(-(r + p) // page)], head)
                k, v = (torch.cat(x)[:r + p] for x in ((k0, k1), (v0, v1)))
                q = state["q"][row:row + r, head * per:(head + 1) * per].double()
                w = q.reshape(r * per, -1) @ k.T.contiguous() / math.sqrt(case["dim"])
                seen = torch.arange(r + p, device="cuda") <= p + torch.arange(r, device="cuda")[:, None]
                w = torch.where(seen.repeat_interleave(per, 0), w, -math.inf).softmax(-1)
                out[row:row + r, head * per:(head + 1) * per] = (w @ v).view(r, per, -1)
                row += r
        s, at = s + len(members), at + sum(r for r, _ in members)
    return out
