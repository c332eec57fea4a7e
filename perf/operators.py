"""The operators of serving with a 4-bit KV cache, as they are measured.

Three families, each in its plain form (elementary torch operations) and as a
user's program calls it (`own`): appending keys and values to the paged 4-bit
cache with the rotation on the way and reading rows back, attention over that
cache, and the log probabilities of given tokens with entropy and top
alternatives.

The cache: pages of 64 positions; [layer][page][KV head] holds one block of K
codes, K scales, V codes, V scales. A row of head_dim values is quantised in
groups of 32: with m the group's value of largest magnitude (the positive one
of a tie), d = m / -8 rounded to 8 significant bits (multiples of 2^-24, at most
8160 in magnitude) is stored as FP16 and each value r as the code
c = clamp(round(r / d), -8, 7) + 8, so that the cache holds d * (c - 8).
Eight consecutive dims are one 32-bit word, the first in the lowest bits. K word
4 j + t (group j) of a row is stored as word t * groups + j; V word n of a block
(counted over all 64 rows) as word n ^ 8 * ((n >> 5) & mask), mask 3 for
head_dim 128 and 1 for 64. K scales lie [position][group], V scales
[position / 2][group][position % 2].
"""
import math
import random

import torch

own = False

PAGE, GROUP = 64, 32
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": 0, "bf16": 1, "f16": 2}


# ---------------------------------------------------------------- the cases

def listed():
    def append(name, type, kv_heads, group, dim, sequences, count, length, ragged, pad, mix):
        return {"name": name, "op": "append", "type": type, "kv_heads": kv_heads, "group": group, "dim": dim,
                "sequences": sequences, "count": count, "length": length, "ragged": ragged, "pad": pad, "mix": mix}

    def attention(name, type, kv_heads, group, dim, sequences, count, length, ragged, pad, mix):
        return dict(append(name, type, kv_heads, group, dim, sequences, count, length, ragged, pad, mix), op="attention")

    def logprobs(name, type, rows, vocab, pad, top, masked):
        return {"name": name, "op": "logprobs", "type": type, "rows": rows, "vocab": vocab, "pad": pad, "top": top,
                "masked": masked}

    return [
        # one session's decode step at the end of the default context: latency
        append("append_decode_1", "f32", 8, 4, 128, 1, 1, 4352, False, 0, 1),
        # one prefill block, the largest the runtime takes
        append("append_block_256", "f32", 8, 4, 128, 1, 256, 4096, False, 0, 2),
        # many sessions' prompts of all lengths in one call, with unused rows behind the last
        append("append_ragged_f16", "f16", 4, 8, 64, 24, 700, 3000, True, 37, 3),
        # a short conversation's next token: latency
        attention("decode_1x500", "f32", 8, 4, 128, 1, 1, 500, False, 0, 4),
        # one session at the default context's end
        attention("decode_1x4352", "f32", 8, 4, 128, 1, 1, 4352, False, 0, 5),
        # a decode step over 64 sessions of all lengths
        attention("decode_64_ragged", "f32", 8, 4, 128, 64, 1, 4352, True, 0, 6),
        # few sessions with very long contexts, more query heads
        attention("decode_4x131072", "bf16", 8, 8, 128, 4, 1, 131072, False, 0, 7),
        # one prefill block behind a long prefix
        attention("block_256_at_4096", "f32", 8, 4, 128, 1, 256, 4352, False, 0, 8),
        # prompts' blocks and decode steps in one call, narrower heads, an odd group
        attention("ragged_mixed_f16", "f16", 4, 5, 64, 24, 230, 3001, True, 19, 9),
        # the last row of a decode step with five alternatives: latency
        logprobs("logprobs_1", "f32", 1, 131072, 0, 5, 0.0),
        # scoring a block of the largest size
        logprobs("logprobs_256", "f32", 256, 131072, 0, 20, 0.0),
        # an odd vocabulary, unaligned rows, half of it ruled out by a grammar
        logprobs("logprobs_odd_bf16", "bf16", 1000, 50001, 2, 8, 0.5),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "logprobs"])
    type = rng.choice(["f32", "bf16", "f16"])
    if kind == "logprobs":
        vocab = _log(rng, 33, 131072)
        rows = _log(rng, 1, max(1, min(4096, 256 * 131072 // vocab)))
        return {"op": kind, "type": type, "rows": rows, "vocab": vocab, "pad": rng.choice([0, 0, 1, 5, 24]),
                "top": rng.randint(0, min(32, vocab)), "masked": rng.choice([0.0, 0.0, 0.3])}
    dim, kv_heads, group = rng.choice([64, 128, 128]), rng.randint(1, 8), rng.randint(1, 8)
    sequences = _log(rng, 1, 64)
    if kind == "append":
        count = _log(rng, 1, max(1, min(1000, 16000 // sequences)))
        length = count + _log(rng, 1, 4000)
    else:
        width = kv_heads * dim
        length = _log(rng, 1, max(1, min(131072, 4 * 131072 * 1024 // (sequences * width))))
        most = 256 * 4352 * 4096 // (sequences * length * width * group)
        count = _log(rng, 1, max(1, min(length, 256, most)))
    return {"op": kind, "type": type, "kv_heads": kv_heads, "group": group, "dim": dim, "sequences": sequences,
            "count": count, "length": length, "ragged": rng.random() < 0.6, "pad": rng.choice([0, 0, 3]),
            "mix": rng.randrange(1 << 30)}


def _shape(case):
    """(rows appended or asked, positions held) of each sequence: the case's maxima for all, or spread
    below them, the first at the maxima, with a sequence without rows now and then."""
    n, most, longest = case["sequences"], case["count"], case["length"]
    if not case["ragged"]:
        return [most] * n, [longest] * n
    rng, counts, lengths = random.Random(case["mix"]), [most], [longest]
    for _ in range(n - 1):
        count = rng.choice([0, 1, 1, _log(rng, 1, most), rng.randint(1, most)]) if most > 1 else int(rng.random() < 0.95)
        counts.append(count)
        lengths.append(max(1, count, _log(rng, max(1, longest // 50), longest)))
    return counts, lengths


def _block_bytes(dim):
    return PAGE * dim + 4 * PAGE * (dim // GROUP)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (16 + 12 * case["top"]), "flops": 5 * n}
    counts, lengths = _shape(case)
    rows, heads, dim = sum(counts), case["kv_heads"], case["dim"]
    row = heads * _block_bytes(dim) // PAGE
    if case["op"] == "append":
        # k, v and q in; the cached rows out and in again; the read rows and the rotated q out
        return {"bytes": rows * (2 * heads * dim * size * 2 + 2 * row + 2 * case["group"] * heads * dim * size),
                "flops": rows * heads * dim * (6 + 3 * case["group"] + 10)}
    seen = sum(c * n - c * (c - 1) // 2 for c, n in zip(counts, lengths))
    held = sum(n for c, n in zip(counts, lengths) if c)
    return {"bytes": held * row + 2 * rows * heads * case["group"] * dim * size,
            "flops": 4 * seen * heads * case["group"] * dim}


# ---------------------------------------------------------------- the inputs

def _rope(positions, dim):
    inverse = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inverse
    angle = torch.cat([angle, angle], 1)
    return angle.cos().float(), angle.sin().float()


def _filled_pool(gen, pages, heads, dim):
    """A pool whose every page holds quantised keys (a few strong channels, as rotated keys have) and values."""
    words, groups = dim // 8, dim // GROUP
    pool = torch.empty((pages, heads, _block_bytes(dim)), dtype=torch.uint8, device="cuda")
    strong = 1 + 2 * (torch.rand((heads, 1, dim), generator=gen, device="cuda") > 0.95).float()
    half = PAGE * dim // 2
    for p0 in range(0, pages, 1024):
        n = min(1024, pages - p0)
        block = pool[p0:p0 + n]
        k = torch.randn((n, heads, PAGE, dim), generator=gen, device="cuda") * strong
        v = torch.randn((n, heads, PAGE, dim), generator=gen, device="cuda")
        codes, d = _quantise(k)
        block[..., :half] = _k_order(_words(codes)).reshape(n, heads, half)
        block[..., half:half + 2 * PAGE * groups] = d.half().reshape(n, heads, -1).view(torch.uint8)
        codes, d = _quantise(v)
        at = _v_words(torch.arange(PAGE * words, device="cuda"), dim)
        order = torch.empty_like(at)
        order[at] = torch.arange(PAGE * words, device="cuda")
        v0 = half + 2 * PAGE * groups
        block[..., v0:v0 + half] = _words(codes).reshape(n, heads, PAGE * words, 4)[:, :, order].reshape(n, heads, half)
        d = d.half().reshape(n, heads, PAGE // 2, 2, groups).transpose(3, 4).reshape(n, heads, -1)
        block[..., v0 + half:] = d.contiguous().view(torch.uint8)
    return pool.reshape(-1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        logits = normal(rows, vocab + case["pad"]) * 2.5
        if case["masked"]:
            logits.masked_fill_(torch.rand(logits.shape, generator=gen, device="cuda") < case["masked"], -math.inf)
            logits[:, 0] = 1.0  # a grammar leaves something
        logits = logits.to(dtype)[:, :vocab]
        targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        top = case["top"]
        return {"case": case, "logits": logits, "targets": targets,
                "logprobs": torch.zeros(rows, device="cuda"), "entropy": torch.zeros(rows, device="cuda"),
                "top_ids": torch.zeros((rows, top), dtype=torch.int64, device="cuda"),
                "top_logprobs": torch.zeros((rows, top), device="cuda")}

    counts, lengths = _shape(case)
    heads, dim, query = case["kv_heads"], case["dim"], case["kv_heads"] * case["group"]
    need = [-(-n // PAGE) for n in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").int()
    table = torch.zeros((len(counts), max(need)), dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    rows = offsets[-1] + case["pad"]
    state = {"case": case, "pages": pages, "rows": rows, "table": table,
             "offsets": torch.tensor(offsets, dtype=torch.int32, device="cuda"),
             "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
    if case["op"] == "attention":
        state["pool"] = _filled_pool(gen, pages, heads, dim)
        state["q"] = (normal(rows, query * dim) * 1.5).to(dtype)
        state["scale"] = 1.0 / math.sqrt(dim)
        state["out"] = torch.zeros((rows, query * dim), dtype=dtype, device="cuda")
        state["workspace"] = None
        return state
    # q | k | v rows as a fused projection leaves them
    state["qkv"] = normal(rows, (query + 2 * heads) * dim).to(dtype)
    state["cos"], state["sin"] = _rope(max(lengths), dim)
    state["pool"] = torch.zeros(pages * heads * _block_bytes(dim), dtype=torch.uint8, device="cuda")
    for name, width in (("q_out", query), ("k_out", heads), ("v_out", heads)):
        state[name] = torch.zeros((rows, width * dim), dtype=dtype, device="cuda")
    return state


# ---------------------------------------------------------------- the plain forms

def _quantise(r):
    """Codes (0..15) and scales of [..., dim] values, in their own precision."""
    g = r.reshape(*r.shape[:-1], -1, GROUP)
    high, low = g.amax(-1), g.amin(-1)
    x = torch.where(high >= -low, high, low) / -8
    unit = torch.ldexp(torch.ones_like(x), (torch.frexp(x).exponent - 8).clamp(min=-24))
    d = (torch.round(x / unit) * unit).clamp(-8160, 8160)
    zero = (d == 0)[..., None]
    c = torch.round(g / torch.where(zero, 1.0, d[..., None])).clamp(-8, 7)
    c = torch.where(zero, 0.0, c)
    return (c + 8).to(torch.uint8).reshape(r.shape), d


def _words(codes):
    """[..., dim] codes -> [..., dim / 8, 4] bytes, two codes each, the earlier dim in the low bits."""
    pairs = codes.reshape(*codes.shape[:-1], codes.shape[-1] // 8, 4, 2)
    return pairs[..., 0] | (pairs[..., 1] << 4)


def _k_order(words):
    """Words 4 j + t of a K row in storage order t * groups + j."""
    *lead, n, four = words.shape
    return words.reshape(*lead, n // 4, 4, four).transpose(-3, -2).reshape(*lead, n, four)


def _v_words(n, dim):
    """Where word n of a block's V codes is stored."""
    return n ^ (8 * ((n >> 5) & (3 if dim == 128 else 1)))


def _values(stored, scales):
    """[..., words, 4] bytes in natural order and [..., groups] scales -> [..., dim] FP32 values."""
    codes = torch.stack([stored & 15, stored >> 4], -1).reshape(*stored.shape[:-2], -1)
    c = codes.float() - 8
    return (c.reshape(*scales.shape, GROUP) * scales.float()[..., None]).reshape(c.shape)


def _row_positions(state):
    """(sequence, position, whether used) of each row."""
    offsets, lengths = state["offsets"].long(), state["lengths"].long()
    row = torch.arange(state["rows"], device="cuda")
    s = torch.searchsorted(offsets, row, right=True) - 1
    used = s < lengths.numel()
    s = s.clamp(max=lengths.numel() - 1)
    return s, (lengths[s] - (offsets[s + 1] - row)).clamp(min=0), used


def _addresses(state, s, position):
    """Byte addresses in the pool of rows' K codes, K scales, V codes and V scales, [rows, heads, bytes]."""
    heads, dim = state["case"]["kv_heads"], state["case"]["dim"]
    words, groups, half = dim // 8, dim // GROUP, PAGE * dim // 2
    page, slot = state["table"].long()[s, position // PAGE], position % PAGE
    head = torch.arange(heads, device="cuda")
    block = ((page[:, None] * heads + head) * _block_bytes(dim))[..., None]
    slot = slot[:, None, None]
    two, byte = torch.arange(2, device="cuda"), torch.arange(4, device="cuda")
    group = torch.arange(groups, device="cuda")
    k = block + slot * (dim // 2) + torch.arange(dim // 2, device="cuda")
    ks = block + half + 2 * slot * groups + torch.arange(2 * groups, device="cuda")
    v0 = half + 2 * PAGE * groups
    n = _v_words(slot * words + torch.arange(words, device="cuda"), dim)
    v = (block[..., None] + v0 + 4 * n[..., None] + byte).flatten(2)
    at = ((slot // 2) * groups + group) * 2 + slot % 2
    vs = (block[..., None] + v0 + half + 2 * at[..., None] + two).flatten(2)
    return k, ks, v, vs


def _rotate(x, cos, sin):
    """Split-half rotation of [rows, heads, dim]; cos and sin [rows, 1, dim]."""
    half = x.shape[-1] // 2
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    return x * cos + turned * sin


def _plain_append(state):
    case = state["case"]
    heads, dim, query = case["kv_heads"], case["dim"], case["kv_heads"] * case["group"]
    s, position, used = _row_positions(state)
    s, position = s[used], position[used]
    dtype = state["qkv"].dtype
    q, k, v = state["qkv"][:s.numel()].split([query * dim, heads * dim, heads * dim], 1)
    q = q.float().reshape(-1, query, dim)
    # 64 bits: a key next to the border between two codes must not fall on the other side
    k, v = k.double().reshape(-1, heads, dim), v.double().reshape(-1, heads, dim)
    cos, sin = state["cos"][position][:, None], state["sin"][position][:, None]
    q = _rotate(q, cos, sin) * (1 + 0.1 * torch.log(1 + (position // 16384).float()))[:, None, None]
    k = _rotate(k, cos.double(), sin.double())
    at_k, at_ks, at_v, at_vs = _addresses(state, s, position)
    pool = state["pool"]
    codes, d = _quantise(k)
    pool[at_k] = _k_order(_words(codes)).flatten(2)
    pool[at_ks] = d.half().contiguous().view(torch.uint8)
    codes, d = _quantise(v)
    pool[at_v] = _words(codes).flatten(2)
    pool[at_vs] = d.half().contiguous().view(torch.uint8)
    # and the rows read back
    rows = s.numel()
    groups, words = dim // GROUP, dim // 8
    k = pool[at_k].reshape(rows, heads, 4, groups, 4).transpose(2, 3).reshape(rows, heads, words, 4)
    k = _values(k, pool[at_ks].contiguous().view(torch.float16))
    v = _values(pool[at_v].reshape(rows, heads, words, 4), pool[at_vs].contiguous().view(torch.float16))
    for name, x in (("q_out", q), ("k_out", k), ("v_out", v)):
        state[name][:rows] = x.reshape(rows, -1).to(dtype)
    return {"q": state["q_out"], "k": state["k_out"], "v": state["v_out"]}


def _plain_attention(state):
    case = state["case"]
    heads, dim, group = case["kv_heads"], case["dim"], case["group"]
    words, groups, half = dim // 8, dim // GROUP, PAGE * dim // 2
    table, offsets, lengths = state["table"].long(), state["offsets"].long(), state["lengths"].long()
    n_seq, n_pages = table.shape
    blocks = state["pool"].reshape(-1, heads, _block_bytes(dim))[table].transpose(1, 2)  # [seq, head, page, bytes]
    lead = (n_seq, heads, n_pages)
    k = blocks[..., :half].reshape(*lead, PAGE, 4, groups, 4).transpose(4, 5).reshape(*lead, PAGE, words, 4)
    ks = blocks[..., half:half + 2 * PAGE * groups].contiguous().view(torch.float16).reshape(*lead, PAGE, groups)
    v0 = half + 2 * PAGE * groups
    at = _v_words(torch.arange(PAGE * words, device="cuda"), dim)
    v = blocks[..., v0:v0 + half].reshape(*lead, PAGE * words, 4)[..., at, :].reshape(*lead, PAGE, words, 4)
    vs = blocks[..., v0 + half:].contiguous().view(torch.float16)
    vs = vs.reshape(*lead, PAGE // 2, groups, 2).transpose(4, 5).reshape(*lead, PAGE, groups)
    k = _values(k, ks).reshape(n_seq, heads, n_pages * PAGE, dim)
    v = _values(v, vs).reshape(n_seq, heads, n_pages * PAGE, dim)
    most = case["count"]
    counts = offsets[1:] - offsets[:-1]
    i = torch.arange(most, device="cuda")
    row = (offsets[:-1, None] + i).clamp(max=state["rows"] - 1)
    q = state["q"][row].float().reshape(n_seq, most, heads, group, dim).permute(0, 2, 3, 1, 4)
    q = q.reshape(n_seq, heads, group * most, dim) * state["scale"]
    scores = q @ k.transpose(2, 3)
    last = lengths[:, None] - counts[:, None] + i                       # position of each row
    seen = torch.arange(n_pages * PAGE, device="cuda") <= last[..., None]  # [seq, row, key]
    scores = scores.reshape(n_seq, heads, group, most, -1).masked_fill_(~seen[:, None, None], -math.inf)
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(n_seq, heads, group * most, -1) @ v).reshape(n_seq, heads, group, most, dim)
    o = (o / torch.where(total == 0, 1.0, total)).permute(0, 3, 1, 2, 4).reshape(n_seq, most, -1)
    live = i < counts[:, None]
    state["out"][row[live]] = o[live].to(state["out"].dtype)
    return state["out"]


def _plain_logprobs(state):
    x, top = state["logits"].float(), state["case"]["top"]
    m = x.amax(1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(1, keepdim=True)
    log_z = torch.log(z)
    shifted = x - m
    entropy = log_z - torch.where(e > 0, e * shifted, 0.0).sum(1, keepdim=True) / z
    out = {"logprobs": (shifted.gather(1, state["targets"][:, None]) - log_z)[:, 0], "entropy": entropy[:, 0]}
    if top:
        # the value's order in the upper half, the id's falling order in the lower: ties go to the lowest id
        bits = (x + 0.0).view(torch.int32)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        ids = torch.arange(x.shape[1], device="cuda")
        keys = order * (1 << 32) + (0xFFFFFFFF - ids)
        out["top_ids"] = 0xFFFFFFFF - (keys.topk(top, 1).values & 0xFFFFFFFF)
        out["top_logprobs"] = shifted.gather(1, out["top_ids"]) - log_z
    return out


# ---------------------------------------------------------------- the framework's operators

def _descriptors(state):
    """The cache's and the rows' descriptors, which a program keeps beside its cache."""
    import lunelette_b200 as L
    case = state["case"]
    cache = L.Kv4(state["pool"].data_ptr(), 1, state["pages"], case["kv_heads"], case["dim"])
    rows = L.Rows(state["rows"], case["sequences"], state["offsets"].data_ptr(), state["lengths"].data_ptr(),
                  state["table"].data_ptr(), state["table"].shape[1], case["count"], case["length"])
    return L.library(), cache, rows


def _own_append(state):
    lib, cache, rows = state["call"]
    case, qkv = state["case"], state["qkv"]
    kind, dim, size = CODES[case["type"]], case["dim"], qkv.element_size()
    query, heads = case["kv_heads"] * case["group"], case["kv_heads"]
    stream, width, q = torch.cuda.current_stream().cuda_stream, qkv.shape[1], qkv.data_ptr()
    k = q + query * dim * size
    v = k + heads * dim * size
    bad = lib.lunelette_cuda_kv4_append(cache, 0, rows, kind, k, width, v, width, q, width, query,
                                        state["q_out"].data_ptr(), query * dim, state["cos"].data_ptr(),
                                        state["sin"].data_ptr(), state["cos"].shape[0], None, stream)
    bad |= lib.lunelette_cuda_kv4_read(cache, 0, rows, kind, state["k_out"].data_ptr(), heads * dim,
                                       state["v_out"].data_ptr(), heads * dim, None, stream)
    if bad:
        raise RuntimeError("append or read was refused")
    return {"q": state["q_out"], "k": state["k_out"], "v": state["v_out"]}


def _own_attention(state):
    lib, cache, rows = state["call"]
    case = state["case"]
    query = case["kv_heads"] * case["group"]
    if state["workspace"] is None:
        need = lib.lunelette_cuda_kv4_attention_workspace(cache, rows, query)
        state["workspace"] = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    width = query * case["dim"]
    if lib.lunelette_cuda_kv4_attention(cache, 0, rows, CODES[case["type"]], state["q"].data_ptr(), width, query,
                                        state["scale"], state["out"].data_ptr(), width,
                                        state["workspace"].data_ptr(), state["workspace"].numel(), None,
                                        torch.cuda.current_stream().cuda_stream):
        raise RuntimeError("attention was refused")
    return state["out"]


def _own_logprobs(state):
    import lunelette_b200 as L
    case, logits, top = state["case"], state["logits"], state["case"]["top"]
    if L.library().lunelette_cuda_token_logprobs(
            logits.data_ptr(), CODES[case["type"]], case["rows"], case["vocab"], logits.stride(0),
            state["targets"].data_ptr(), top, state["logprobs"].data_ptr(), state["entropy"].data_ptr(),
            state["top_ids"].data_ptr() if top else None, state["top_logprobs"].data_ptr() if top else None,
            torch.cuda.current_stream().cuda_stream):
        raise RuntimeError("token_logprobs was refused")
    out = {"logprobs": state["logprobs"], "entropy": state["entropy"]}
    if top:
        out.update(top_ids=state["top_ids"], top_logprobs=state["top_logprobs"])
    return out


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"append": _plain_append, "attention": _plain_attention, "logprobs": _plain_logprobs}[op](state)
    if op == "logprobs":
        return _own_logprobs(state)
    if "call" not in state:
        state["call"] = _descriptors(state)
    return _own_append(state) if op == "append" else _own_attention(state)


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_values(state, sequence, length, kind):
    """[heads, length, dim] values of one sequence's keys (kind 0) or values (1), each by its own address."""
    heads, dim = state["case"]["kv_heads"], state["case"]["dim"]
    groups, half = dim // GROUP, PAGE * dim // 2
    p = torch.arange(length, device="cuda")[None, :, None]
    d = torch.arange(dim, device="cuda")[None, None]
    h = torch.arange(heads, device="cuda")[:, None, None]
    page, slot = state["table"][sequence].long()[p // PAGE], p % PAGE
    base = (page * heads + h) * _block_bytes(dim)
    if kind == 0:
        word = slot * (dim // 8) + (d % 32 // 8) * groups + d // 32
        scale = base + half + 2 * (slot * groups + d // 32)
    else:
        line = (slot * dim + d) // 256  # 32 words of 8 codes
        word = slot * (dim // 8) + d // 8
        word = word ^ ((line % (4 if dim == 128 else 2)) << 3)
        base = base + half + 2 * PAGE * groups
        scale = base + half + 2 * ((slot // 2) * 2 * groups + (d // 32) * 2 + slot % 2)
    pool = state["pool"]
    codes = (pool[base + 4 * word + d % 8 // 2].long() >> (4 * (d % 2))) % 16
    bits = pool[scale].to(torch.int32) + 256 * pool[scale + 1].to(torch.int32)
    return (codes - 8).double() * bits.to(torch.int16).view(torch.float16).double()


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "logprobs":
        out = {"logprobs": [], "entropy": [], "top_ids": [], "top_logprobs": []}
        for x, t in zip(state["logits"].split(64), state["targets"].split(64)):
            logp = torch.log_softmax(x.double(), 1)
            p = logp.exp()
            out["logprobs"].append(logp[torch.arange(len(t), device="cuda"), t])
            out["entropy"].append(torch.special.entr(p).sum(1))
            if case["top"]:
                ids = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :case["top"]]
                out["top_ids"].append(ids)
                out["top_logprobs"].append(torch.take_along_dim(logp, ids, 1))
        return {k: torch.cat(v) for k, v in out.items() if v}
    counts, lengths = _shape(case)
    heads, dim, group = case["kv_heads"], case["dim"], case["group"]
    if case["op"] == "attention":
        out = torch.zeros((state["rows"], heads * group, dim), dtype=torch.float64, device="cuda")
        first = 0
        for s, (count, length) in enumerate(zip(counts, lengths)):
            if count:
                k, v = (_exact_values(state, s, length, kind) for kind in (0, 1))
                q = state["q"][first:first + count].double().reshape(count, heads, group, dim)
                scores = torch.einsum("chgd,hnd->hgcn", q, k) / math.sqrt(dim)
                hidden = torch.ones((count, length), dtype=torch.bool, device="cuda").triu(length - count + 1)
                p = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
                out[first:first + count] = torch.einsum("hgcn,hnd->chgd", p, v).reshape(count, heads * group, dim)
            first += count
        return out.reshape(state["rows"], -1)
    out = {name: torch.zeros((state["rows"], n * dim), dtype=torch.float64, device="cuda")
           for name, n in (("q", heads * group), ("k", heads), ("v", heads))}
    position = torch.cat([torch.arange(n - c, n, device="cuda") for c, n in zip(counts, lengths)])
    rows = position.numel()
    x = state["qkv"][:rows].double().reshape(rows, -1, 2, dim // 2)
    cos = state["cos"][position].double()[:, None, :dim // 2]
    sin = state["sin"][position].double()[:, None, :dim // 2]
    a, b = x[:, :, 0], x[:, :, 1]
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    query = heads * group
    stretch = 1 + 0.1 * torch.log1p(torch.div(position, 16384, rounding_mode="floor").double())
    out["q"][:rows] = (turned[:, :query] * stretch[:, None, None]).flatten(1)
    for name, r in (("k", turned[:, query:query + heads]), ("v", x[:, query + heads:].flatten(2))):
        g = r.reshape(rows, -1, GROUP)
        most = g.abs().amax(-1, keepdim=True)
        m = torch.where((g == most).any(-1, keepdim=True), most, -most)
        # 8 significant bits of m / -8, on the grid of FP16's smallest step
        step = torch.clamp(torch.exp2(torch.floor(torch.log2(most / 8)) - 7), min=2.0 ** -24)
        d = torch.clamp(torch.round(m / -8 / step) * step, -8160, 8160)
        c = torch.where(d == 0, 0.0, torch.clamp(torch.round(g / d), -8, 7))
        out[name][:rows] = (c * d).reshape(rows, -1)
    return out
