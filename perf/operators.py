"""Performance cases of the paged 4-bit KV cache and the rotary embedding that
goes with it: what a program that serves several long contexts at once calls
for each attention layer.

Kinds (`kind` of a case):
  rope    ops.bind_rope: query rows rotated at their positions;
  append  ops.bind_paged_append, then ops.bind_paged_read of the same rows:
          new keys (rotated on the way) and values put into the 4-bit pages of
          their sequences, and the rows as the cache now holds them;
  attend  ops.bind_paged_gqa: causal attention of every sequence's rows over
          its pages.

A pool is bytes [pages, kv_heads, page / 32, 40 * dim]: one block of 32 keys
of one KV head is 40 * dim bytes, laid out as _block_bytes() says.

Heads are the repository's (16 query / 4 KV heads of 256) and the 64 and 128
wide ones of its tests.
"""
import math

import torch

own = False

THETA = 1e7
LIMIT = 16384.0  # values are kept to +-LIMIT


def listed():
    return [
        # the query heads of one decoded token: the smallest call
        rope("rope_decode", 1, 262_131, 16, 256, 64, "half", "none"),
        # a prompt of a model with interleaved pairs over the whole head, its
        # context stretched
        rope("rope_prompt_2k", 2048, 30_000, 16, 128, 128, "interleaved", "yarn"),
        # a large batch of prompts, part of the head rotated
        rope("rope_prompt_16k", 16381, 0, 16, 256, 64, "half", "linear"),
        # one token for each of some chats
        append("append_decode_16", 16, 1, 8191, 4, 256, 64, 64, "half"),
        # a chunk of one long prompt
        append("append_chunk_2k", 1, 2048, 2048, 4, 256, 64, 128, "half"),
        # prompts of many lengths that start at odd places of their pages
        append("append_ragged", 13, 901, 4099, 8, 128, 128, 32, "interleaved"),
        # a token of a chat at a medium context: the smallest attention
        attend("attend_decode_4k", 1, 1, 4096, 16, 4, 256, 64),
        # a token of a long document, at no round length
        attend("attend_decode_32k", 1, 1, 32749, 16, 4, 256, 64),
        # a token for each of many chats of many lengths
        attend("attend_batch_48", 48, 1, 16384, 16, 4, 256, 32),
        # the next message of a conversation: a short chunk, a long history
        attend("attend_turn_16k", 1, 61, 16411, 16, 4, 256, 128),
        # a large chunk of a long prompt
        attend("attend_chunk_2k", 1, 2048, 2048, 16, 4, 256, 64),
        # several messages of odd lengths at once, eight query heads a KV head
        attend("attend_ragged", 7, 517, 3001, 32, 4, 128, 32),
    ]


def _named(name, case):
    return case if name is None else {"name": name, **case}


def rope(name, tokens, first, heads, dim, rotary, layout, scaling):
    return _named(name, {"kind": "rope", "tokens": tokens, "first": first, "heads": heads, "dim": dim,
                         "rotary": rotary, "layout": layout, "scaling": scaling})


def append(name, sequences, rows, past, kv_heads, dim, rotary, page, layout):
    return _named(name, {"kind": "append", "sequences": sequences, "rows": rows, "past": past,
                         "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "page": page,
                         "layout": layout})


def attend(name, sequences, rows, past, q_heads, kv_heads, dim, page):
    return _named(name, {"kind": "attend", "sequences": sequences, "rows": rows, "past": past,
                         "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page})


def _log(rng, low, high):
    """A whole number from low to high, spread evenly over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choices(["rope", "append", "attend"], [20, 25, 55])[0]
    dim = rng.choice([256, 256, 128, 64])
    layout = rng.choice(["half", "interleaved"])
    rotary = rng.choice([dim, dim // 2, dim // 4, 2 * rng.randint(1, dim // 2)])
    if kind == "rope":
        heads = rng.choice([4, 8, 16, 32])
        tokens = _log(rng, 1, 16384 * 4096 // (heads * dim))
        return rope(None, tokens, _log(rng, 1, 1_000_000) - 1, heads, dim, rotary, layout,
                    rng.choice(["none", "linear", "yarn"]))
    kv_heads, page = rng.choice([1, 2, 4, 8]), rng.choice([32, 64, 128, 256])
    if kind == "append":
        sequences = _log(rng, 1, 32)
        rows = 1 if rng.random() < 0.3 else _log(rng, 1, 2048 * 4 * 256 // (sequences * kv_heads * dim) + 1)
        return append(None, sequences, rows, _log(rng, 1, 8192) - 1, kv_heads, dim, rotary, page, layout)
    group = rng.choice([1, 2, 4, 4, 5, 8, 16])
    while group * kv_heads > 32:
        group = (group + 1) // 2
    if rng.random() < 0.5:  # single tokens: the cache's bytes at most the largest listed batch's
        sequences = _log(rng, 1, 48)
        past = _log(rng, 1, min(65536, 48 * 16384 * 1024 // (2 * sequences * kv_heads * dim)))
        return attend(None, sequences, 1, past, group * kv_heads, kv_heads, dim, page)
    sequences = _log(rng, 1, 8)
    pairs = 2048 * 2048 * 4096 // (sequences * group * kv_heads * dim)  # half the largest chunk's work
    rows = _log(rng, 2, min(2048, math.isqrt(pairs)))
    past = _log(rng, 1, min(32768, max(1, pairs // rows - rows))) - 1
    return attend(None, sequences, rows, past, group * kv_heads, kv_heads, dim, page)


# ---------------------------------------------------------------- lengths

def _lengths(case):
    """(rows, past) of each sequence: the first has the case's own, the others
    between an eighth of them and all."""
    rows, past = [case["rows"]], [case["past"]]
    for s in range(1, case["sequences"]):
        rows.append(max(1, case["rows"] * (2 + (s * 37 + 5) % 13) // 16))
        past.append(case["past"] * (2 + (s * 53 + 11) % 15) // 16)
    return rows, past


def frequencies(rotary, scaling):
    """(frequencies fp32, factor) of a rotation: theta^(-2i / rotary), divided
    by 4 (linear), or by 8 where a pair turns less than once over 32768
    positions, with a ramp up to 32 turns (yarn)."""
    f = THETA ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    factor = 1.0
    if scaling == "linear":
        f = f / 4.0
    elif scaling == "yarn":
        turns = 32768 * f / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        f, factor = f * keep + f / 8.0 * (1 - keep), 0.1 * math.log(8.0) + 1.0
    return f.float(), torch.tensor(factor, dtype=torch.float32).item()


# ----------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rows16(g, *shape):
    """Activations: normal, with a few channels of every head that are larger."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    large = 1 + 4 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.03).float()
    return (x * large).half()


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] == "rope":
        freqs, factor = frequencies(case["rotary"], case["scaling"])
        first = case["first"] + int(seed) % 7
        return {"case": case, "x": _rows16(g, case["tokens"], case["heads"], case["dim"]),
                "positions": torch.arange(first, first + case["tokens"], dtype=torch.int32, device="cuda"),
                "freqs": freqs.cuda(), "factor": factor,
                "out": torch.empty(case["tokens"], case["heads"], case["dim"], dtype=torch.float16,
                                   device="cuda")}
    rows, past = _lengths(case)
    dim, hkv, page, total = case["dim"], case["kv_heads"], case["page"], sum(rows)
    state = {"case": case, "total": total, "most_rows": max(rows),
             "most_keys": max(r + p for r, p in zip(rows, past)),
             "starts": torch.tensor([0] + rows).cumsum(0).int().cuda(),
             "past": torch.tensor(past, dtype=torch.int32).cuda()}
    # every sequence's pages, anywhere in a pool that has some more
    need = [-(-(r + p) // page) for r, p in zip(rows, past)]
    order = torch.randperm(sum(need) + 3, generator=g, device="cuda").int()
    table = torch.zeros(len(need), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    state["table"] = table
    pool = torch.zeros(sum(need) + 3, hkv, page // 32, 40 * dim, dtype=torch.uint8, device="cuda")
    if case["kind"] == "append":
        freqs, factor = frequencies(case["rotary"], "none")
        state |= {"pool": pool, "freqs": freqs.cuda(), "factor": factor}
        state |= {n: _rows16(g, total, hkv, dim) for n in ("k", "v")}
        state |= {n: torch.empty_like(state[n[0]]) for n in ("k_out", "v_out")}
        return state
    state["pool"] = _filled(pool, g, dim)
    state["q"] = _rows16(g, total, case["q_heads"], dim)
    state["out"] = torch.empty_like(state["q"])
    return state


def _filled(pool, g, dim):
    """The pool with every block holding 32 keys and values."""
    flat = pool.view(-1, 40 * dim)
    for at in range(0, flat.shape[0], 4096):
        part = flat[at:at + 4096]
        k, v = (_quantized(_rows16(g, part.shape[0], 32, dim)) for _ in range(2))
        part.copy_(_block_bytes(*k, *v))
    return pool


# ------------------------------------------------------- the 4-bit format

def _quantized(x):
    """(codes, scale, bias) of groups of 32 channels: x fp16 [..., dim]."""
    x = x.float().nan_to_num(0.0, LIMIT, -LIMIT).clamp(-LIMIT, LIMIT)
    x = x.unflatten(-1, (-1, 32))
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


def _lane_channels(dim):
    return 32 if dim >= 128 else 16


def _block_bytes(kc, ks, kb, vc, vs, vb):
    """Blocks [n, 40 dim] of the keys' and values' codes [n, 32, groups, 32]
    and scales and biases [n, 32, groups]."""
    n, _, groups, _ = kc.shape
    dim, lane = 32 * groups, _lane_channels(32 * groups)
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
    lane, groups = _lane_channels(dim), dim // 32
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


def _block_values(data):
    """K and V fp16 [n, 32, dim] of blocks [n, 40 dim]."""
    k, ks, kb, v, vs, vb = _block_parts(data)
    return _values(k, ks, kb), _values(v, vs, vb)


# ------------------------------------------------------------- plain forms

def run(state):
    if own:
        return _run_own(state)
    return {"rope": _plain_rope, "append": _plain_append, "attend": _plain_attend}[
        state["case"]["kind"]](state)


def _rotated(x, positions, freqs, factor, layout):
    """fp16 rows [T, H, dim] rotated at positions [T], in fp32."""
    angle = positions.double()[:, None] * freqs.double()
    c, s = (angle.cos() * factor).float()[:, None], (angle.sin() * factor).float()[:, None]
    half = freqs.numel()
    rot, rest = x[..., :2 * half].float(), x[..., 2 * half:]
    pairs = rot.unflatten(-1, (2, half) if layout == "half" else (half, 2))
    axis = -2 if layout == "half" else -1
    a, b = pairs.unbind(axis)
    turned = torch.stack((a * c - b * s, b * c + a * s), axis).flatten(-2)
    return torch.cat((turned.half(), rest), -1)


def _plain_rope(state):
    return _rotated(state["x"], state["positions"], state["freqs"], state["factor"],
                    state["case"]["layout"])


def _row_places(state):
    """(sequence, position) of every row of the call."""
    row = torch.arange(state["total"], device="cuda")
    seq = torch.searchsorted(state["starts"][1:], row, right=True)
    return seq, state["past"][seq].long() + row - state["starts"][seq]


def _plain_append(state):
    case, pool = state["case"], state["pool"]
    seq, pos = _row_places(state)
    k = _rotated(state["k"], pos, state["freqs"], state["factor"], case["layout"])
    new = [*_quantized(k), *_quantized(state["v"])]
    # the blocks that the rows lie in, with the rows put in their places
    page, dim = case["page"], case["dim"]
    block = state["table"][seq, pos // page].long() * (page // 32) + pos % page // 32
    touched, at = torch.unique(block, return_inverse=True)
    blocks = pool.view(-1, case["kv_heads"], page // 32, 40 * dim)
    where = (touched // (page // 32), slice(None), touched % (page // 32))
    old = _block_parts(blocks[where].flatten(0, 1))
    for part, rows in zip(old, new):
        part.view(touched.numel(), case["kv_heads"], *part.shape[1:])[at, :, pos % 32] = rows
    blocks[where] = _block_bytes(*old).view(touched.numel(), case["kv_heads"], -1)
    k, v = (x.view(-1, case["kv_heads"], 32, dim)[at, :, pos % 32]
            for x in _block_values(blocks[where].flatten(0, 1)))
    return {"k": k, "v": v}


def _plain_attend(state):
    case = state["case"]
    page, dim, hkv = case["page"], case["dim"], case["kv_heads"]
    seqs, most_rows, most_keys = case["sequences"], state["most_rows"], state["most_keys"]
    group = case["q_heads"] // hkv
    # every sequence's keys and values, padded to the longest
    blocks = state["pool"][state["table"].long()].transpose(2, 3)  # [S, pages, blocks, Hkv, bytes]
    width = blocks.shape[1] * page
    k, v = (x.view(seqs, width // 32, hkv, 32, dim).transpose(1, 2).reshape(seqs, hkv, width, dim)
            [:, :, :most_keys].float() for x in _block_values(blocks.reshape(-1, 40 * dim)))
    # the query rows likewise
    seq, pos = _row_places(state)
    row = torch.arange(state["total"], device="cuda") - state["starts"][seq]
    q = torch.zeros(seqs, most_rows, hkv, group, dim, device="cuda")
    q[seq, row] = state["q"].view(-1, hkv, group, dim).float()
    q = q.permute(0, 2, 1, 3, 4).flatten(2, 3)
    scores = q @ k.transpose(-1, -2).contiguous() / math.sqrt(dim)
    last = state["past"][:, None] + torch.arange(most_rows, device="cuda")
    hidden = torch.arange(most_keys, device="cuda") > last.repeat_interleave(group, 1)[..., None]
    scores.masked_fill_(hidden[:, None], -torch.inf)
    scores = (scores - scores.amax(-1, keepdim=True)).exp()
    out = (scores @ v) / scores.sum(-1, keepdim=True)
    out = out.unflatten(2, (most_rows, group)).permute(0, 2, 1, 3, 4)[seq, row]
    return out.reshape(state["total"], case["q_heads"], dim).half()


# ------------------------------------------------------- the framework's

def _run_own(state):
    from llminfer_amd import ops

    kind = state["case"]["kind"]
    if "calls" not in state:  # bound once, as a serving loop keeps them
        if kind == "rope":
            state["calls"] = [ops.bind_rope(state["x"], state["positions"], state["freqs"], state["out"],
                                            layout=state["case"]["layout"], factor=state["factor"])]
        else:
            place = (state["starts"], state["past"], state["table"])
            if kind == "append":
                state["calls"] = [
                    ops.bind_paged_append(state["k"], state["v"], state["pool"], *place,
                                          freqs=state["freqs"], layout=state["case"]["layout"],
                                          factor=state["factor"]),
                    ops.bind_paged_read(state["pool"], *place, state["k_out"], state["v_out"])]
            else:
                state["calls"] = [ops.bind_paged_gqa(state["q"], state["pool"], *place, state["out"])]
    for call in state["calls"]:
        call()
    return {"k": state["k_out"], "v": state["v_out"]} if kind == "append" else state["out"]


# ------------------------------------------------------------------- work

def work(case):
    if case["kind"] == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": n * case["dim"] * 4 + case["tokens"] * 4, "flops": n * case["rotary"] * 3}
    rows, past = _lengths(case)
    n = case["kv_heads"] * case["dim"]
    if case["kind"] == "append":
        # rows read, packed, and returned as the cache holds them
        return {"bytes": sum(rows) * n * (4 + 1.25 + 4), "flops": sum(rows) * n * 2 * 10}
    keys = sum(r + p for r, p in zip(rows, past))
    pairs = sum(r * p + r * (r + 1) // 2 for r, p in zip(rows, past))
    heads = case["q_heads"] * case["dim"]
    return {"bytes": keys * n * 1.25 + sum(rows) * heads * 4, "flops": 4 * heads * pairs}


# ------------------------------------------------- the definitions, 64 bits

def _place64(key, channel, dim):
    """Where a block keeps (byte, shift) the code and (byte) the scale of a
    key's and of a value's channel; biases are 2 and 64 bytes further."""
    m, t, h, v = key >> 4, key >> 3 & 1, key >> 2 & 1, key & 3
    per = 32 if dim >= 128 else 16
    group = channel >> 5
    nib = channel % 8 // 2 + channel % 2 * 4
    lane = channel // per % 4 * 16 + 8 * m + 4 * h + v
    k_at = t * 8 * dim + channel // (4 * per) * 32 * per + lane * (per // 2) + channel % per // 8 * 4
    k_scale = 16 * dim + t * 2 * dim + (group * 16 + 8 * m + 4 * h + v) * 4
    slot = 4 * t + v
    vnib = slot // 2 + slot % 2 * 4
    v_at = 20 * dim + channel // 64 * 1024 + ((2 * m + h) * 16 + channel % 16) * 16 + channel // 16 % 4 * 4
    v_scale = 36 * dim + group * 128 + ((2 * m + h) * 8 + slot) * 2
    return k_at + nib // 2, nib % 2 * 4, k_scale, v_at + vnib // 2, vnib % 2 * 4, v_scale


def _cached64(state, s, head, count):
    """K and V of a sequence's first keys, one KV head, by the definition."""
    case = state["case"]
    dim, page = case["dim"], case["page"]
    key = torch.arange(count, device="cuda")[:, None]
    channel = torch.arange(dim, device="cuda")[None]
    pages = state["table"][s].long()[key // page]
    base = ((pages * case["kv_heads"] + head) * (page // 32) + key % page // 32) * (40 * dim)
    data, halves = state["pool"].view(-1), state["pool"].view(-1).view(torch.float16)
    k_at, k_shift, k_scale, v_at, v_shift, v_scale = _place64(key % 32, channel, dim)

    def value(at, shift, scale, bias):
        code = (data[base + at] >> shift.to(torch.uint8)) & 15
        x = (16 + code.double()) * halves[(base + scale) // 2].double()
        return (x + halves[(base + bias) // 2].double()).half().double()

    return (value(k_at, k_shift.expand(count, dim), k_scale, k_scale + 2),
            value(v_at, v_shift.expand(count, dim), v_scale, v_scale + 64))


def _turned64(x, positions, freqs, factor, layout):
    x, half = x.double(), freqs.numel()
    phase = torch.polar(torch.full((), factor, dtype=torch.float64, device="cuda"),
                        positions.double()[:, None] * freqs.double())[:, None]
    first = torch.arange(half, device="cuda") * (1 if layout == "half" else 2)
    second = first + (half if layout == "half" else 1)
    z = torch.complex(x[..., first], x[..., second]) * phase
    x[..., first], x[..., second] = z.real, z.imag
    return x


def _kept64(x):
    """The values that the cache keeps of fp16 rows."""
    x = x.double().clamp(-LIMIT, LIMIT).unflatten(-1, (-1, 32))
    low = x.amin(-1, keepdim=True)
    s = ((x.amax(-1, keepdim=True) - low) / 15).half().double()
    b = (low - 16 * s).half().double()
    code = torch.where(s > 0, (x - b) / s, 16.0).round().clamp(16, 31)
    return (code * s + b).half().double().flatten(-2)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rope":
        return _turned64(state["x"], state["positions"], state["freqs"], state["factor"], case["layout"])
    rows, past = _lengths(case)
    if case["kind"] == "append":
        positions = torch.cat([torch.arange(p, p + r) for r, p in zip(rows, past)]).cuda()
        k = _turned64(state["k"], positions, state["freqs"], state["factor"], case["layout"]).half()
        return {"k": _kept64(k), "v": _kept64(state["v"])}
    group = case["q_heads"] // case["kv_heads"]
    out = torch.empty(state["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for s, (r, p) in enumerate(zip(rows, past)):
        seen = torch.arange(r + p, device="cuda") <= p + torch.arange(r, device="cuda")[:, None]
        for head in range(case["kv_heads"]):
            k, v = _cached64(state, s, head, r + p)
            for h in range(head * group, (head + 1) * group):
                w = state["q"][at:at + r, h].double() @ k.T.contiguous() / math.sqrt(case["dim"])
                w = torch.where(seen, w, -math.inf).softmax(-1)
                out[at:at + r, h] = w @ v
        at += r
    return out

