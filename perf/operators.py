"""The serving operators next to the Qwen2 step, as cases to measure: a paged key/value cache held in 4 bits
(append, attention, moving its pages) and the log probabilities of a step's tokens.

``own`` chooses between the operators' plain forms, written here in elementary torch operations, and the
framework's kernels (``nanocompile_b200.serving``). Both read the same state: the packed cache, its page table,
the rows. ``exact`` computes a case in 64 bits, apart from both.

The cache, as every function here reads it. A page holds ``page`` positions (a multiple of 16) of one layer as
``page / 16`` tiles for each key/value head: [head][tile][20 * d bytes]. A tile is 16 positions: key codes
(8 d bytes), key parameters (2 d), value codes (8 d), value parameters (2 d). Values are quantised in blocks of
32 along the head dimension: zero = f16(min), scale = f16((max - min) * f32(1/15)), code = clamp(floor((x - zero)
* (1 / scale) + 1/2), 0, 15) (0 where the scale is 0), and stand for zero + scale * code. With position t = 8 j + g = 8 j + 2 c + h of its tile,
block b, VB = 2 blocks at a time where their number is even and else 1:
  key codes     u32 word [b / VB][g][c][b % VB][j]: nibble i is dimension 32 b + 8 c + i
  value codes   u32 word [b / VB][g][c][b % VB][j]: half-word h, nibble i is dimension 32 b + 4 g + i
  parameters    u32 word [g][b][j]: scale in the low half-word, zero in the high one (f16)
"""

import math
import random

import numpy as np
import torch

own = False

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
CUDA = "cuda"


# -- the cases ---------------------------------------------------------------------------------------------


def listed():
    return [
        # One chat of the 0.5B model, early on: one new token over 97 cached positions. Latency decides.
        attention("decode-one-97", "float32", 14, 2, 64, seqs=1, kv=97, rows=1),
        # The batched decode of the benchmark: 64 sequences with 2048 cached positions each.
        attention("decode-64x2048", "float32", 14, 2, 64, seqs=64, kv=2048, rows=1),
        # A serving batch of a larger model with long, ragged histories and one idle slot.
        attention("decode-ragged-24x16k", "bfloat16", 32, 8, 128, seqs=24, kv=16384, rows=1, ragged=True),
        # The 512-token prompt of the benchmark, attended once it is in the cache.
        attention("prompt-512", "float32", 14, 2, 64, seqs=1, kv=512, rows=512),
        # The next chunks of two long prompts, over what their earlier chunks left in the cache.
        attention("chunk-2x1000-of-6001", "bfloat16", 32, 8, 128, seqs=2, kv=6001, rows=1000),
        # A decode step's new keys and values for 13 sequences, rotated, quantised and read back.
        append("append-13", "float32", 2, 64, seqs=13, kv=700, rows=1, ragged=True),
        # A prompt's keys and values, 4 x 2048 rows.
        append("append-4x2048", "bfloat16", 8, 128, seqs=4, kv=2048, rows=2048),
        # A step of beam search: 8 beams of 211 positions take over one another's histories, each one longer.
        pages("beam-step-8", "update", seqs=8, kv=211, page_bytes=24 * 2 * 64 * 64 * 5 // 4, page=64, beams=8),
        # 64 prompts in 256 slots of a server, each forked into four samples; their last pages are copied.
        pages("fork-64-to-256", "update", seqs=256, kv=4096, page_bytes=24 * 2 * 64 * 64 * 5 // 4, page=64, beams=4),
        # A server's pool, half of whose sequences have left, packed.
        pages("compact-64", "compact", seqs=64, kv=4000, page_bytes=24 * 2 * 16 * 64 * 5 // 4, page=16, beams=1),
        # Token scores of one decode step: the chosen token, the entropy, five alternatives.
        logprobs("logprobs-1", "float32", 1, 151936, targets=1, top=5),
        # The scores of a 512-token prompt's tokens with twenty alternatives, some of the vocabulary masked.
        logprobs("logprobs-512", "float32", 512, 151936, targets=1, top=20, masked=True),
    ]


def attention(name, dtype, heads, kv_heads, d, seqs, kv, rows, ragged=False, page=64):
    return {"name": name, "kind": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "d": d,
            "seqs": seqs, "kv": kv, "rows": rows, "ragged": ragged, "page": page}


def append(name, dtype, kv_heads, d, seqs, kv, rows, ragged=False, page=64):
    return {"name": name, "kind": "append", "dtype": dtype, "kv_heads": kv_heads, "d": d, "seqs": seqs, "kv": kv,
            "rows": rows, "ragged": ragged, "page": page}


def pages(name, kind, seqs, kv, page_bytes, page, beams):
    return {"name": name, "kind": kind, "seqs": seqs, "kv": kv, "page_bytes": page_bytes, "page": page, "beams": beams}


def logprobs(name, dtype, rows, vocab, targets, top, masked=False):
    return {"name": name, "kind": "logprobs", "dtype": dtype, "rows": rows, "vocab": vocab, "targets": targets,
            "top": top, "masked": masked}


def draw(rng):
    """One more case of the same ranges: sizes spread over their logarithms, odd ones among them."""

    def size(low, high):
        return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))

    kind = rng.choice(["decode", "decode", "prompt", "append", "update", "compact", "logprobs", "logprobs"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    heads, kv_heads, d = rng.choice([(14, 2, 64), (2, 1, 64), (4, 2, 32), (32, 8, 128), (12, 12, 96), (64, 4, 128),
                                     (16, 16, 64), (6, 2, 96)])
    page = rng.choice([16, 32, 64, 128])
    if kind == "decode":
        kv = size(1, 32768)
        seqs = size(1, max(1, min(128, 24 * 16384 * 8 * 128 // (kv * kv_heads * d))))
        case = attention("", dtype, heads, kv_heads, d, seqs, kv, 1, rng.random() < 0.6, page)
    elif kind == "prompt":
        rows = size(2, 1024)
        kv = rows + rng.choice([0, size(1, 5000)])
        seqs = size(1, max(1, min(16, 2 * 1000 * 6001 * 32 * 128 // (rows * kv * heads * d))))
        case = attention("", dtype, heads, kv_heads, d, seqs, kv, rows, rng.random() < 0.5, page)
    elif kind == "append":
        rows = size(1, 2048)
        seqs = size(1, max(1, min(64, 4 * 2048 * 8 * 128 // (rows * kv_heads * d))))
        case = append("", dtype, kv_heads, d, seqs, rows + size(1, 2048), rows, rng.random() < 0.5, page)
    elif kind in ("update", "compact"):
        beams = rng.choice([1, 2, 4, 8])
        kv = size(1, 4096)
        seqs = beams * size(1, min(256, (64 * 4096 // kv) // (1 if kind == "update" else beams)) // beams or 1)
        case = pages("", kind, seqs, kv, size(1, 24) * 2 * page * 64 * 5 // 4, page, beams)
    else:
        rows = size(1, 512)
        case = logprobs("", dtype, rows, size(32, 151936), rng.choice([0, 1, 1, 4]), rng.choice([0, 1, 5, 20, 32]),
                        rng.random() < 0.3)
    del case["name"]
    return case


# -- what a case's rows look like: made on the host from the seed -------------------------------------------


def sequences(case, seed):
    """The lengths of the case's sequences (after this step's rows) and how many rows each of them has."""
    rng = random.Random("%d %r" % (seed, sorted((k, v) for k, v in case.items() if k != "name")))
    n, kv, rows = case["seqs"], case["kv"], case["rows"]
    if not case["ragged"]:
        return [kv] * n, [rows] * n
    counts = [rows if rows == 1 else rng.randint(max(1, rows // 4), rows) for _ in range(n)]
    lengths = [rng.randint(max(c, kv // 8), kv) for c in counts]
    counts[0], lengths[0] = rows, kv
    if rows == 1 and n > 2:
        lengths[n // 2] = 0                     # an idle slot of the batch: its row sees nothing
    return lengths, counts


def bench_lengths(case):
    """The mean lengths that `work` counts with: sequences()' own, whatever the seed, by their expectation."""
    if not case["ragged"]:
        return case["seqs"] * case["kv"], case["seqs"] * case["rows"]
    n = case["seqs"]
    rows = 1 if case["rows"] == 1 else 0.625 * case["rows"]
    idle = 1 if case["rows"] == 1 and n > 2 else 0
    return case["kv"] + max(0, n - 1 - idle) * 0.5625 * case["kv"], case["rows"] + (n - 1) * rows


def rotation(positions, d, base=1e6):
    """cos and sin of RoPE's angles, float32 [positions, d / 2]."""
    rates = 1.0 / base ** (torch.arange(0, d, 2, device=CUDA, dtype=torch.float32) / d)
    angles = torch.arange(positions, device=CUDA, dtype=torch.float32)[:, None] * rates
    return torch.cos(angles).contiguous(), torch.sin(angles).contiguous()


def prepare(case, seed):
    g = torch.Generator(device=CUDA).manual_seed(seed)
    kind = case["kind"]
    if kind in ("attention", "append"):
        return prepare_cache(case, seed, g)
    if kind in ("update", "compact"):
        return prepare_pages(case, seed, g)
    rows, vocab = case["rows"], case["vocab"]
    # Logits as a language model gives them: a broad bulk and a few tokens well above it.
    logits = torch.randn(rows, vocab, device=CUDA, generator=g) * 2.0
    peaks = torch.randint(0, vocab, (rows, min(8, vocab)), device=CUDA, generator=g)
    logits.scatter_add_(1, peaks, torch.rand(peaks.shape, device=CUDA, generator=g) * 12)
    if case["masked"]:                                         # a constrained step: part of the vocabulary is out
        logits[:, torch.rand(vocab, device=CUDA, generator=g) < 0.25] = -math.inf
    targets = torch.randint(0, vocab, (rows, case["targets"]), device=CUDA, generator=g)
    if case["targets"]:
        targets[:, 0] = torch.where(torch.rand(rows, device=CUDA, generator=g) < 0.7, peaks[:, 0], targets[:, 0])
    state = {"case": case, "logits": logits.to(TYPES[case["dtype"]]), "targets": targets}
    if own:
        from nanocompile_b200 import serving

        state["scratch"] = torch.zeros(serving.token_logprobs_scratch_bytes(rows, vocab, case["top"]), device=CUDA,
                                       dtype=torch.uint8)
    return state


def prepare_cache(case, seed, g):
    lengths, counts = sequences(case, seed)
    kv_heads, d, page, n = case["kv_heads"], case["d"], case["page"], case["seqs"]
    width = max(1, -(-case["kv"] // page))
    needed = [-(-m // page) for m in lengths]
    total = sum(needed)
    count = total + total // 8 + 1
    # The pages of a server that has run for a while lie anywhere in its pool.
    order = torch.randperm(count, device=CUDA, generator=g).to(torch.int32)
    held = torch.arange(width, device=CUDA)[None] < torch.tensor(needed, device=CUDA)[:, None]
    table = torch.full((n, width), -1, device=CUDA, dtype=torch.int32)
    table[held] = order[:total]
    dtype = TYPES[case["dtype"]]
    kept = [m if case["kind"] == "attention" else max(0, m - c) for m, c in zip(lengths, counts)]
    # What is not held by a sequence is what earlier ones left there: any bytes.
    pool = torch.randint(0, 256, (count, kv_heads * page * d * 5 // 4), device=CUDA, generator=g, dtype=torch.uint8)
    bias = torch.randn(kv_heads, d, device=CUDA, generator=g) * (torch.rand(kv_heads, d, device=CUDA, generator=g) < 0.1) * 4
    fill(pool, table, kept, bias, g, page, kv_heads, d)
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = int(starts[-1])
    state = {"case": case, "pool": pool, "table": table, "lengths": torch.tensor(lengths, device=CUDA, dtype=torch.int32),
             "row_start": torch.tensor(starts, device=CUDA, dtype=torch.int32), "rope": rotation(max(1, case["kv"]), d),
             "max_rows": max(counts)}
    if case["kind"] == "attention":
        # q, k and v come out of one projection: the queries are a strided part of its rows.
        qkv = torch.randn(rows, (case["heads"] + 2 * kv_heads) * d, device=CUDA, generator=g).to(dtype)
        state["q"] = qkv[:, : case["heads"] * d]
        state["out"] = torch.empty(rows, case["heads"] * d, device=CUDA, dtype=dtype)
    else:
        kvs = torch.randn(rows, 2 * kv_heads * d, device=CUDA, generator=g)
        kvs[:, : kv_heads * d] += bias.reshape(-1)
        kvs = kvs.to(dtype)
        state["keys"], state["values"] = kvs[:, : kv_heads * d], kvs[:, kv_heads * d:]
    if own:
        from nanocompile_b200 import serving

        state["layout"] = layout = serving.KV4Layout(case.get("heads", kv_heads), kv_heads, d, page)
        if case["kind"] == "attention":
            size = serving.kv4_attention_scratch_bytes(layout, rows, n, case["kv"], state["max_rows"])
            state["scratch"] = torch.zeros(size, device=CUDA, dtype=torch.uint8)
    return state


def fill(pool, table, kept, bias, g, page, kv_heads, d):
    """Quantised keys and values N(0, 1) (the keys with a few channels off centre) for each sequence's kept positions."""
    at, tile = page // 16, 20 * d
    view = pool.view(-1, kv_heads, at, tile)
    for i, m in enumerate(kept):
        if m == 0:
            continue
        have = -(-m // 16)
        x = torch.randn(2, have * 16, kv_heads, d, device=CUDA, generator=g)
        x[0] += bias
        codes, scale, zero = quantise(x)
        tiles = pack(codes, scale, zero)                                  # [have, kv_heads, tile]
        where = table[i].long().repeat_interleave(at)[:have], torch.arange(have, device=CUDA) % at
        view[where[0], :, where[1]] = tiles


def prepare_pages(case, seed, g):
    rng = random.Random("%d %r" % (seed, sorted((k, v) for k, v in case.items() if k != "name")))
    n, kv, page, beams = case["seqs"], case["kv"], case["page"], case["beams"]
    width = -(-(kv + 8) // page)
    update = case["kind"] == "update"
    # Groups of `beams` slots share their history up to where they parted, as an earlier fork left them.
    table = np.full((n, width), -1, np.int32)
    lengths = np.zeros(n, np.int32)
    entries, fork = [], update and n > beams
    for first in range(0, n, beams):
        length = kv if first == 0 else rng.randint(max(1, kv // 2), kv)
        parted = rng.randint(0, length) // page
        for i in range(first, first + beams):
            if (fork and i > first) or (not update and i > 0 and rng.random() < 0.5):
                continue                                                 # an empty slot
            held = -(-length // page)
            shared = parted if i > first and lengths[first] else 0
            table[i, :shared] = table[first, :shared]
            entries += [(i, j) for j in range(shared, held)]
            table[i, shared:held] = np.arange(len(entries) - (held - shared), len(entries))
            lengths[i] = length
    used = len(entries)
    # The pool has room for every slot's history without sharing, whatever the seed.
    count = (n // beams if fork else n) * -(-kv // page) + 2 * n
    order = np.array(rng.sample(range(count), used), np.int32) if used else np.zeros(0, np.int32)
    table = np.where(table >= 0, order[np.maximum(table, 0)] if used else table, -1).astype(np.int32)
    if fork:                                                              # every sample of a prompt from its first slot
        parent = np.array([i - i % beams for i in range(n)], np.int32)
    else:                                                                 # a beam step, within each group
        parent = np.array([i - i % beams + rng.randrange(beams) for i in range(n)], np.int32)
    grow = np.ones(n, np.int32)
    put = lambda a: torch.from_numpy(a).to(CUDA)                          # noqa: E731
    pool = torch.randint(0, 256, (count, case["page_bytes"]), device=CUDA, generator=g, dtype=torch.uint8)
    state = {"case": case, "pool": pool, "table": put(table), "lengths": put(lengths), "parent": put(parent),
             "grow": put(grow), "new_table": torch.empty(n, width, device=CUDA, dtype=torch.int32),
             "new_lengths": torch.empty(n, device=CUDA, dtype=torch.int32),
             "status": torch.zeros(4, device=CUDA, dtype=torch.int64)}
    if own:
        from nanocompile_b200 import serving

        state["scratch"] = torch.zeros(serving.kv_pages_scratch_bytes(n, width, count), device=CUDA, dtype=torch.uint8)
    return state


# -- one pass ------------------------------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attention": own_attention, "append": own_append, "update": own_update, "compact": own_compact,
                "logprobs": own_logprobs}[kind](state)
    return {"attention": plain_attention, "append": plain_append, "update": plain_update, "compact": plain_compact,
            "logprobs": plain_logprobs}[kind](state)


def stream():
    return torch.cuda.current_stream().cuda_stream


def own_attention(state):
    from nanocompile_b200 import serving

    serving.kv4_attention(state["layout"], state["out"], state["q"], state["pool"], state["table"], state["lengths"],
                          state["scratch"], max_length=state["case"]["kv"], row_start=state["row_start"],
                          max_rows=state["max_rows"], rope=state["rope"], stream=stream())
    return state["out"]


def own_append(state):
    from nanocompile_b200 import serving

    at = stream()
    serving.kv4_append(state["layout"], state["pool"], state["keys"], state["values"], state["table"], state["lengths"],
                       row_start=state["row_start"], rope=state["rope"], stream=at)
    keys, values = (torch.empty_like(state[k], dtype=torch.float32, memory_format=torch.contiguous_format)
                    for k in ("keys", "values"))
    serving.kv4_read(state["layout"], keys, values, state["pool"], state["table"], state["lengths"],
                     row_start=state["row_start"], stream=at)
    return keys, values


def own_update(state):
    from nanocompile_b200 import serving

    serving.kv_pages_update(state["new_table"], state["new_lengths"], state["table"], state["lengths"], state["pool"],
                            state["status"], state["scratch"], page_size=state["case"]["page"], parent=state["parent"],
                            grow=state["grow"], stream=stream())
    return state["new_table"], state["new_lengths"], state["status"], state["pool"]


def own_compact(state):
    from nanocompile_b200 import serving

    serving.kv_pages_compact(state["new_table"], state["table"], state["lengths"], state["pool"], state["status"],
                             state["scratch"], page_size=state["case"]["page"], stream=stream())
    return state["new_table"], state["status"], state["pool"]


def own_logprobs(state):
    from nanocompile_b200 import serving

    case, rows = state["case"], state["case"]["rows"]
    out = torch.empty(rows, case["targets"], device=CUDA)
    entropy = torch.empty(rows, device=CUDA)
    top = torch.empty(rows, case["top"], device=CUDA, dtype=torch.int64)
    top_logprobs = torch.empty(rows, case["top"], device=CUDA)
    serving.token_logprobs(state["logits"], state["targets"], out, entropy, top, top_logprobs, scratch=state["scratch"],
                           stream=stream())
    return out, entropy, top, top_logprobs


# -- the plain forms -------------------------------------------------------------------------------------------


def quantise(x):
    """Codes, scale and zero (f16) of blocks of 32 of the last dimension, in 32 bits."""
    x = x.reshape(*x.shape[:-1], -1, 32)
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    limit = 65504.0
    zero = low.clamp(-limit, limit).half()
    scale = ((high - low) * torch.full_like(low, 1 / 15)).clamp(max=limit).half()
    s = scale.float()
    codes = torch.floor((x - zero.float()) * (torch.ones_like(s) / torch.where(s > 0, s, 1.0)) + 0.5).clamp(0, 15)
    return torch.where(s > 0, codes, 0.0).to(torch.int32), scale[..., 0], zero[..., 0]


def pack(codes, scale, zero):
    """[2, 16 tiles, heads, blocks, 32] codes and their parameters to the bytes of tiles, [tiles, heads, 20 d]."""
    _, t, heads, nb, _ = codes.shape
    tiles, vb = t // 16, 2 - nb % 2
    shift = torch.arange(8, device=codes.device, dtype=torch.int32) * 4
    k = (codes[0].view(tiles, 2, 8, heads, nb // vb, vb, 4, 8) << shift).sum(-1, dtype=torch.int64)   # T j g H B v c
    k = k.permute(0, 3, 4, 2, 6, 5, 1)                                                     # T H B g c v j
    v = (codes[1].view(tiles, 2, 4, 2, heads, nb // vb, vb, 8, 4) << shift[:4]).sum(-1, dtype=torch.int64)  # T j c h H B v g
    v = (v[:, :, :, 0] | v[:, :, :, 1] << 16).permute(0, 3, 4, 6, 2, 5, 1)                   # T H B g c v j
    par = scale.contiguous().view(torch.int16).long() & 0xFFFF | (zero.contiguous().view(torch.int16).long() & 0xFFFF) << 16
    par = par.view(2, tiles, 2, 8, heads, nb).permute(0, 1, 4, 3, 5, 2)                      # 2 T H g b j
    words = [w.reshape(tiles, heads, -1) for w in (k, par[0], v, par[1])]
    low32 = torch.cat(words, -1)
    return torch.where(low32 >= 2**31, low32 - 2**32, low32).to(torch.int32).view(torch.uint8)


def unpack(tiles, d):
    """[n, heads, page / 16, 20 d] bytes to the keys and values they stand for, [2, n, page, heads, d] float32."""
    n, heads, at, _ = tiles.shape
    nb = d // 32
    vb = 2 - nb % 2
    words = tiles.contiguous().view(torch.int32)
    shift = torch.arange(8, device=tiles.device, dtype=torch.int32) * 4
    k, kp, v, vp = words.split([2 * d, d // 2, 2 * d, d // 2], -1)
    k = k.reshape(n, heads, at, nb // vb, 8, 4, vb, 2, 1) >> shift & 15                       # n H T B g c v j i
    k = k.permute(0, 2, 7, 4, 1, 3, 6, 5, 8).reshape(n, at * 16, heads, nb, 32)
    v = v.reshape(n, heads, at, nb // vb, 8, 4, vb, 2, 1, 1) >> (shift[:4] + shift[4:5] * torch.arange(2, device=v.device)[:, None].int()) & 15
    v = v.permute(0, 2, 7, 5, 8, 1, 3, 6, 4, 9).reshape(n, at * 16, heads, nb, 32)            # n T j c h H B v g i
    par = torch.stack([kp, vp]).reshape(2, n, heads, at, 8, nb, 2).contiguous().view(torch.float16)
    par = par.view(2, n, heads, at, 8, nb, 2, 2).permute(0, 1, 3, 6, 4, 2, 5, 7).reshape(2, n, at * 16, heads, nb, 2).float()
    codes = torch.stack([k, v])
    return (par[..., 1:] + par[..., :1] * codes).reshape(2, n, at * 16, heads, d)


def rows_of(state):
    """Each row's sequence and position."""
    start, lengths = state["row_start"].long(), state["lengths"].long()
    rows = torch.arange(state.get("q", state.get("keys")).shape[0], device=CUDA)
    seq = torch.searchsorted(start, rows, right=True) - 1
    return seq, lengths[seq] - (start[seq + 1] - rows)


def rotate(x, position, rope):
    """x [rows, heads, d] in 32 bits, rotated by its rows' positions; each product and sum rounded by itself."""
    cos, sin = (t[position.clamp(min=0)][:, None] for t in rope)
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def plain_attention(state):
    case = state["case"]
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["d"], case["page"]
    n, width = state["table"].shape
    q = state["q"].float().view(-1, heads, d)
    seq, position = rows_of(state)
    q = rotate(q, position, state["rope"])
    most, kv = state["max_rows"], width * page
    slot = torch.arange(q.shape[0], device=CUDA) - state["row_start"].long()[seq]
    padded = q.new_zeros(n, most, heads, d)
    padded[seq, slot] = q
    at = torch.full((n, most), -1, device=CUDA)
    at[seq, slot] = position
    tiles = state["pool"].view(-1, kv_heads, page // 16, 20 * d)[state["table"].clamp(min=0).long().flatten()]
    keys, values = unpack(tiles, d).view(2, n, kv, kv_heads, d)
    held = torch.arange(kv, device=CUDA) < state["lengths"][:, None]                        # [n, kv]
    keys, values = (torch.where(held[:, :, None, None], x, 0.0) for x in (keys, values))
    grouped = padded.view(n, most, kv_heads, heads // kv_heads, d).permute(0, 2, 3, 1, 4).flatten(2, 3)   # n H (G r) d
    scores = grouped @ keys.permute(0, 2, 3, 1) * d ** -0.5
    seen = (torch.arange(kv, device=CUDA) <= at[:, :, None])[:, None, None]                 # n 1 1 r kv
    scores = torch.where(seen, scores.view(n, kv_heads, -1, most, kv), -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = weights.sum(-1, keepdim=True)
    out = weights.flatten(2, 3) @ values.permute(0, 2, 1, 3)
    out = out.view(n, kv_heads, -1, most, d) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, most, heads * d)[seq, slot]
    return out.to(state["q"].dtype)


def plain_append(state):
    case = state["case"]
    kv_heads, d, page = case["kv_heads"], case["d"], case["page"]
    seq, position = rows_of(state)
    keys = rotate(state["keys"].float().view(-1, kv_heads, d), position, state["rope"])
    values = state["values"].float().view(-1, kv_heads, d)
    codes, scale, zero = quantise(torch.stack([keys, values]))                               # 2 r H nb (32)
    ok = position >= 0
    seq, position, codes, scale, zero = seq[ok], position[ok], codes[:, ok], scale[:, ok], zero[:, ok]
    nb = d // 32
    vb = 2 - nb % 2
    block = state["table"][seq, position // page].long()[:, None, None]
    t = position % 16
    j, g, c, h = (x[:, None, None] for x in (t // 8, t % 8, t % 8 // 2, t % 2))
    head = torch.arange(kv_heads, device=CUDA)[None, :, None]
    b = torch.arange(nb, device=CUDA)[None, None]
    base = block * state["pool"].shape[1] + ((head * (page // 16) + (position % page // 16)[:, None, None]) * 20 * d)
    shift = torch.arange(8, device=CUDA, dtype=torch.int32) * 4
    # key words: [b / vb][g][c][b % vb][j]
    word = (codes[0].view(-1, kv_heads, nb, 4, 8) << shift).sum(-1, dtype=torch.int64)       # r H nb 4
    chunk = torch.arange(4, device=CUDA)
    at = base[..., None] // 4 + (((b // vb * 8 + g)[..., None] * 4 + chunk) * vb + (b % vb)[..., None]) * 2 + j[..., None]
    pool32, pool16 = state["pool"].view(torch.int32).view(-1), state["pool"].view(torch.int16).view(-1)
    pool32[at.flatten()] = torch.where(word >= 2**31, word - 2**32, word).to(torch.int32).flatten()
    # value half-words
    half = (codes[1].view(-1, kv_heads, nb, 8, 4) << shift[:4]).sum(-1, dtype=torch.int64)    # r H nb 8
    group = torch.arange(8, device=CUDA)
    at = (base[..., None] + 10 * d) // 2 + ((((b // vb * 8)[..., None] + group) * 4 + c[..., None]) * vb * 2
                                             + ((b % vb) * 2 + j)[..., None]) * 2 + h[..., None]
    pool16[at.flatten()] = torch.where(half >= 2**15, half - 2**16, half).to(torch.int16).flatten()
    # parameters: [g][b][j]
    at = (base + 8 * d) // 2 + ((g * nb + b) * 2 + j) * 2
    pool16[at.flatten()] = scale[0].contiguous().view(torch.int16).flatten()
    pool16[at.flatten() + 1] = zero[0].contiguous().view(torch.int16).flatten()
    pool16[at.flatten() + 5 * d] = scale[1].contiguous().view(torch.int16).flatten()
    pool16[at.flatten() + 5 * d + 1] = zero[1].contiguous().view(torch.int16).flatten()
    # what the rows now hold, read back
    out = torch.zeros(2, ok.shape[0], kv_heads, d, device=CUDA)
    tiles = state["pool"].view(-1, kv_heads, page // 16, 20 * d)[block[:, 0, 0], :, position % page // 16]
    read = unpack(tiles[:, :, None], d)                                                      # 2 r 16 H d
    out[:, ok] = read[:, torch.arange(t.shape[0], device=CUDA), t]
    return out[0].flatten(1), out[1].flatten(1)


def plain_update(state):
    page, old, pool = state["case"]["page"], state["table"], state["pool"]
    n, width = old.shape
    count = pool.shape[0]
    parent = state["parent"].long()
    none = parent < 0
    before = torch.where(none, 0, state["lengths"][parent.clamp(min=0)].long())
    after = torch.where(none, 0, (before + state["grow"]).clamp(0, width * page))
    kept = torch.minimum(before, after)
    column = torch.arange(width, device=CUDA)
    taken = torch.where(column < ((kept + page - 1) // page)[:, None], old[parent.clamp(min=0)].long(), -1)
    # A last page that is not full belongs to one sequence: the first that would write to it, if no other reads past there.
    tail = kept // page
    partial = (kept % page != 0) & (after > 0)
    tail_page = torch.where(partial, taken.gather(1, tail.clamp(max=width - 1)[:, None])[:, 0], count)
    refs = torch.zeros(count + 1, device=CUDA, dtype=torch.int64)
    refs.scatter_add_(0, torch.where(taken >= 0, taken, count).flatten(), torch.ones(n * width, device=CUDA, dtype=torch.int64))
    tails = torch.zeros(count + 1, device=CUDA, dtype=torch.int64).scatter_add_(0, tail_page, torch.ones(n, device=CUDA, dtype=torch.int64))
    index = torch.arange(n, device=CUDA)
    owner = torch.full((count + 1,), n, device=CUDA).scatter_reduce_(0, tail_page, index, "amin")
    copied = partial & ~((refs[tail_page] == tails[tail_page]) & (owner[tail_page] == index))
    fresh = torch.where(copied, tail, (kept + page - 1) // page)
    need = (column >= fresh[:, None]) & (column < ((after + page - 1) // page)[:, None])
    # Kept references only: a copied tail no longer refers to its source, which another sequence holds.
    free = (refs[:count] == 0).nonzero()[:, 0]
    wanted = int(need.sum())
    short = max(0, wanted - free.shape[0])
    if short:
        used = torch.unique(old[(column < ((state["lengths"].long() + page - 1) // page)[:, None]) & (old >= 0)]).shape[0]
        return old.clone(), state["lengths"].clone(), torch.tensor([short, used, 0, 0], device=CUDA), pool
    new = taken.clone()
    new[need] = free[:wanted]
    source, target = taken.gather(1, tail.clamp(max=width - 1)[:, None])[:, 0][copied], new.gather(1, tail.clamp(max=width - 1)[:, None])[:, 0][copied]
    pool[target] = pool[source]
    used = int((refs[:count] > 0).sum()) + wanted
    status = torch.tensor([0, used, int(copied.sum()), int(new.max()) + 1], device=CUDA)
    return new.to(torch.int32), after.to(torch.int32), status, pool


def plain_compact(state):
    page, old, pool = state["case"]["page"], state["table"].long(), state["pool"]
    n, width = old.shape
    count = pool.shape[0]
    column = torch.arange(width, device=CUDA)
    live = (column < ((state["lengths"].long() + page - 1) // page)[:, None]) & (old >= 0)
    seen = torch.zeros(count, device=CUDA, dtype=torch.bool)
    seen[old[live]] = True
    used = int(seen.sum())
    holes, high = (~seen[:used]).nonzero()[:, 0], seen[used:].nonzero()[:, 0] + used
    moved = torch.arange(count, device=CUDA)
    moved[high] = holes
    pool[holes] = pool[high]
    new = torch.where(live, moved[old.clamp(min=0)], -1)
    return new.to(torch.int32), torch.tensor([0, used, holes.shape[0], used], device=CUDA), pool


def plain_logprobs(state):
    case, x = state["case"], state["logits"].float()
    top = x.amax(-1, keepdim=True)
    centred = x - top
    e = torch.exp(centred)
    total = e.sum(-1)
    log_total = torch.log(total)
    entropy = log_total - torch.where(e > 0, e * centred, 0.0).sum(-1) / total
    out = centred.gather(1, state["targets"]) - log_total[:, None]
    # The largest logits, the lowest index first among equals: one whole number orders both.
    bits = x.view(torch.int32).long() & 0xFFFFFFFF
    bits = torch.where(x == 0, 0, bits)
    order = torch.where(bits >= 2**31, 2**32 - 1 - bits, bits + 2**31) - 2**31
    key = order * 2**32 + (2**32 - 1 - torch.arange(x.shape[1], device=CUDA))
    ids = 2**32 - 1 - (torch.topk(key, case["top"], dim=-1).values & 0xFFFFFFFF)
    return out, entropy, ids, centred.gather(1, ids) - log_total[:, None]


# -- what a pass cannot do without -----------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind in ("attention", "append"):
        size = 4 if case["dtype"] == "float32" else 2
        positions, rows = bench_lengths(case)
        line = case["kv_heads"] * case["d"] * 2 * 5 / 8                   # a position's keys and values in the cache
        table = 4 * positions / case["page"]
        if kind == "append":
            own_bytes = rows * case["kv_heads"] * case["d"] * 2
            return {"bytes": int(rows * line * 2 + own_bytes * (size + 4) + table), "flops": int(12 * own_bytes)}
        seen = positions - rows / 2 * (case["rows"] - 1) / max(1, case["rows"]) if case["rows"] > 1 else positions
        pairs = seen if case["rows"] == 1 else rows * max(1.0, positions / case["seqs"] - rows / case["seqs"] / 2)
        return {"bytes": int(positions * line + 2 * rows * case["heads"] * case["d"] * size + table),
                "flops": int(4 * pairs * case["heads"] * case["d"])}
    if kind in ("update", "compact"):
        n, kv, beams = case["seqs"], case["kv"], case["beams"]
        held = 0.75 * kv / case["page"]
        table = 8 * n * (kv + 8) / case["page"]
        if kind == "update":
            fork = n > beams
            copies = n * (beams - 1) / beams if fork else n * (1 - (1 - (1 - 1 / beams) ** beams)) if beams > 1 else 0
            return {"bytes": int(table + 2 * copies * case["page_bytes"] + 16 * n), "flops": 0}
        moves = 0.25 * held * (1 + (n - 1) / 2)
        return {"bytes": int(table + 2 * moves * case["page_bytes"] + 8 * n), "flops": 0}
    size = 4 if case["dtype"] == "float32" else 2
    rows, vocab = case["rows"], case["vocab"]
    return {"bytes": int(rows * (vocab * size + case["targets"] * 12 + 4 + case["top"] * 12)), "flops": int(6 * rows * vocab)}


# -- the definition, in 64 bits ----------------------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "logprobs":
        return exact_logprobs(case, state)
    if kind == "attention":
        return exact_attention(case, state, seed)
    if kind == "append":
        return exact_append(case, state, seed)
    return None


def exact_logprobs(case, state):
    """A row at a time: the stable order of the logits, and sums in 64 bits."""
    rows = case["rows"]
    if rows * case["vocab"] > 1 << 27:
        return None
    out, entropy, ids, best = [], [], [], []
    for r in range(rows):
        x = state["logits"][r].double()
        p = torch.softmax(x, -1)
        logp = x - torch.logsumexp(x, -1)
        entropy.append(-(p * torch.where(p > 0, logp, 0.0)).sum())
        out.append(logp[state["targets"][r]])
        order = torch.sort(x, descending=True, stable=True).indices[: case["top"]]
        ids.append(order)
        best.append(logp[order])
    return torch.stack(out), torch.stack(entropy), torch.stack(ids), torch.stack(best)


def positions_held(case, state, length, pages):
    """The keys and values of a sequence's first `length` positions, decoded byte by byte: [2, length, heads, d]."""
    kv_heads, d, page = case["kv_heads"], case["d"], case["page"]
    nb = d // 32
    vb = 2 if nb % 2 == 0 else 1
    raw = state["pool"][torch.tensor(pages, device=CUDA).long()].view(len(pages), kv_heads, page // 16, 20 * d)
    t = torch.arange(length, device=CUDA)
    tiles = raw[t // page, :, t % page // 16]                              # [length, heads, 20 d]
    j, g, c, h = t % 16 // 8, t % 8, t % 8 // 2, t % 2

    def byte(at):
        return torch.gather(tiles, 2, at[:, None, None].expand(-1, kv_heads, 1))[..., 0].long()

    def half(at):
        return (byte(at) | byte(at + 1) << 8).to(torch.int16).view(torch.float16).double()

    both = torch.empty(2, length, kv_heads, d, device=CUDA, dtype=torch.float64)
    for b in range(nb):
        for which in range(2):
            at = 8 * d + 10 * d * which + ((g * nb + b) * 2 + j) * 4
            scale, zero = half(at), half(at + 2)
            for i in range(32):
                if which == 0:
                    word = (((b // vb * 8 + g) * 4 + i // 8) * vb + b % vb) * 2 + j
                    place = word * 4 + i % 8 // 2
                else:
                    word = (((b // vb * 8 + i // 4) * 4 + c) * vb + b % vb) * 2 + j
                    place = 10 * d + word * 4 + h * 2 + i % 4 // 2
                both[which, :, :, 32 * b + i] = zero + scale * (byte(place) >> (4 * (i % 2)) & 15)
    return both


def exact_attention(case, state, seed):
    heads, kv_heads, d, page = case["heads"], case["kv_heads"], case["d"], case["page"]
    lengths, counts = sequences(case, seed)
    if sum(lengths) * kv_heads * d > 1 << 29 or sum(c * m for c, m in zip(counts, lengths)) * heads > 1 << 30:
        return None
    table, outs, at = state["table"].cpu().numpy(), [], 0
    cos, sin = (t.double() for t in state["rope"])
    for i, (m, count) in enumerate(zip(lengths, counts)):
        q = state["q"][at: at + count].double().view(count, heads, d)
        at += count
        if m == 0:
            outs.append(torch.zeros(count, heads * d, device=CUDA, dtype=torch.float64))
            continue
        keys, values = positions_held(case, state, m, table[i][: -(-m // page)])
        p = torch.arange(m - count, m, device=CUDA)
        a, b = q[..., : d // 2], q[..., d // 2:]
        u, w = cos[p][:, None], sin[p][:, None]
        q = torch.cat([a * u - b * w, b * u + a * w], -1)
        mask = torch.arange(m, device=CUDA)[None] > p[:, None]
        per = []
        for x in range(heads):
            scores = (q[:, x] @ keys[:, x // (heads // kv_heads)].T) / math.sqrt(d)
            per.append(torch.softmax(scores.masked_fill(mask, -math.inf), -1) @ values[:, x // (heads // kv_heads)])
        outs.append(torch.stack(per, 1).reshape(count, heads * d))
    return torch.cat(outs)


def exact_append(case, state, seed):
    """The values that the quantised rows stand for. The rounding steps (f32 rotation, f16 parameters) are the definition's."""
    kv_heads, d = case["kv_heads"], case["d"]
    lengths, counts = sequences(case, seed)
    where = np.concatenate([np.arange(m - c, m) for m, c in zip(lengths, counts)])
    cos, sin = (t.cpu().numpy()[np.maximum(where, 0)][:, None] for t in state["rope"])
    done = []
    for name in ("keys", "values"):
        x = state[name].float().cpu().numpy().reshape(-1, kv_heads, d)
        if name == "keys":
            a, b = x[..., : d // 2], x[..., d // 2:]
            x = np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)
        x = x.reshape(x.shape[0], kv_heads, d // 32, 32)
        low, high = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
        zero, scale = low.astype(np.float16), ((high - low) * np.float32(1 / 15)).astype(np.float16)
        s = np.where(scale > 0, scale, 1).astype(np.float32)
        code = np.clip(np.floor((x - zero.astype(np.float32)) * (np.float32(1) / s) + np.float32(0.5)), 0, 15) * (scale > 0)
        held = (zero.astype(np.float64) + scale.astype(np.float64) * code).reshape(x.shape[0], -1)
        held[where < 0] = 0
        done.append(torch.from_numpy(held).to(CUDA))
    return tuple(done)
