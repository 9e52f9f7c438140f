"""What the requests of a batch have of their own, as cases to measure: low-rank adapters beside the shared projections, and
beam search's selection and reordering of states.

``own`` chooses between the operators' plain forms, written here in elementary torch operations, and the framework's
kernels (``nanocompile_b200.serving``). Both read the same state. ``exact`` computes a case in 64 bits, apart from both.

Adapters. A row r of sequence i with adapter a gets, for output n of target t (q, k and v are three targets that share x),

    out[r, n] = base[r, n] + scale[a] * sum_j b[a, n, j] * (sum_k a[a, t * rank + j, k] * x[r, k]),   j < ranks[a],

and a row of a sequence without one (-1) is base[r]. ``a``: [slots, targets * rank, inputs], ``b``: [slots, outputs, rank].

Beams. Request g has rows g * beams .. of logits, a score each (the sum of its tokens' log probabilities; -inf: no beam).
A live beam's candidates are score + log softmax(logits); a finished one goes on as itself, with the token ``end``. The best
``beams`` of a request's candidates, divided by their beam's ``norms`` where there are any, go on; among equals the lower beam,
then the lower token.

States. new[i, :, p] = old[parent[i], :, p] for the parent's positions, and at their end one position more.
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
        # One chat of the 0.5B model with an adapter on q, k and v: one new token. Latency decides.
        lora("lora-decode-1", "float32", "bfloat16", 896, (896, 128, 128), 16, slots=8, adapters=1, seqs=1, rows=1),
        # The batched decode of the benchmark, 64 requests; adapters of different ranks on the down projection, every
        # eighth request without one. The batch has just changed, so its rows are grouped anew.
        lora("lora-decode-64-ranks", "float32", "float16", 4864, (896,), 64, slots=100, adapters=24, seqs=64, rows=1, none=8,
             mixed_ranks=True, fresh=True),
        # A larger model's decode step, every request with an adapter of its own: the adapters' bytes bound it.
        lora("lora-decode-128-own", "bfloat16", "bfloat16", 4096, (4096,), 64, slots=128, adapters=128, seqs=128, rows=1),
        # The 512-token prompt of the benchmark through q, k and v.
        lora("lora-prompt-512", "float32", "bfloat16", 896, (896, 128, 128), 16, slots=8, adapters=1, seqs=1, rows=512),
        # Prompts of a larger model, 8 of up to 1024 tokens with 5 adapters, q, k and v.
        lora("lora-prompts-8x1024", "bfloat16", "bfloat16", 4096, (4096, 1024, 1024), 32, slots=16, adapters=5, seqs=8, rows=1024,
             ragged=True),
        # The first choice of one request's 4 beams.
        beams("beams-1x4", "float32", 1, 4, 151936),
        # A batch of 32 requests with 8 beams each; some have ended, part of the vocabulary is out, longer ones count less.
        beams("beams-32x8", "float32", 32, 8, 151936, finished=True, masked=True, norms=True),
        # 48 requests with 16 beams, logits in 16 bits.
        beams("beams-48x16-bf16", "bfloat16", 48, 16, 50257, finished=True),
        # The float32 cache of the 0.5B model's decode step (24 layers, keys and values of 2 heads), 8 beams of 211 positions.
        reorder("reorder-cache-8x211", "float32", groups=1, beams=8, planes=96, capacity=256, length=211, inner=64),
        # The same of 8 requests with 4 beams, up to 2000 positions.
        reorder("reorder-cache-32x2000", "float32", groups=8, beams=4, planes=96, capacity=2048, length=2000, inner=64),
        # Token histories of 64 requests with 4 beams.
        reorder("reorder-tokens-256", "int64", groups=64, beams=4, planes=1, capacity=2048, length=777, inner=1),
    ]


def lora(name, dtype, wtype, inputs, widths, rank, slots, adapters, seqs, rows, none=0, mixed_ranks=False, ragged=False, fresh=False):
    """`adapters` of the `slots` are in use; every `none`-th sequence has none; `fresh`: the rows are grouped in the pass."""
    return {"name": name, "kind": "lora", "dtype": dtype, "wtype": wtype, "inputs": inputs, "widths": "+".join(map(str, widths)),
            "rank": rank, "slots": slots, "adapters": adapters, "seqs": seqs, "rows": rows, "none": none,
            "mixed_ranks": mixed_ranks, "ragged": ragged, "fresh": fresh}


def beams(name, dtype, groups, width, vocab, finished=False, masked=False, norms=False):
    return {"name": name, "kind": "beams", "dtype": dtype, "groups": groups, "beams": width, "vocab": vocab,
            "finished": finished, "masked": masked, "norms": norms}


def reorder(name, dtype, groups, beams, planes, capacity, length, inner):
    return {"name": name, "kind": "reorder", "dtype": dtype, "groups": groups, "beams": beams, "planes": planes,
            "capacity": capacity, "length": length, "inner": inner}


def draw(rng):
    """One more case of the same ranges: sizes spread over their logarithms, odd ones among them."""

    def size(low, high):
        return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))))

    kind = rng.choice(["decode", "decode", "decode", "prompt", "prompt", "beams", "beams", "beams", "reorder", "tokens"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    if kind in ("decode", "prompt"):
        wtype = rng.choice(["float16", "bfloat16"]) if dtype == "float32" else dtype
        inputs, widths = rng.choice([(896, (896, 128, 128)), (896, (896,)), (896, (4864, 4864)), (4864, (896,)), (64, (64, 32, 32)),
                                     (4096, (4096, 1024, 1024)), (4096, (4096,)), (1000, (333,)), (2048, (2048, 515))])
        rank = rng.choice([8, 16, 32, 64])
        if kind == "decode":
            seqs, rows = size(1, 128), 1
        else:
            rows = size(2, 1024)
            seqs = size(1, max(1, min(8, 8 * 1024 * 4096 // (rows * max(inputs, sum(widths))))))
        adapters = size(1, seqs)
        case = lora("", dtype, wtype, inputs, widths, rank, slots=adapters + rng.choice([0, 0, size(1, 20)]), adapters=adapters,
                    seqs=seqs, rows=rows, none=rng.choice([0, 0, 3, 8]) if seqs > adapters else 0, mixed_ranks=rng.random() < 0.4,
                    ragged=rows > 1 and rng.random() < 0.5, fresh=rng.random() < 0.4)
    elif kind == "beams":
        vocab, width = size(32, 151936), rng.choice([1, 2, 3, 4, 5, 8, 16, 32])
        case = beams("", dtype, size(1, max(1, min(64, 256 * 151936 // (vocab * width)))), width, vocab, rng.random() < 0.4,
                     rng.random() < 0.3, rng.random() < 0.3)
    elif kind == "reorder":
        capacity = size(16, 2048)
        width = rng.choice([1, 2, 4, 5, 8])
        planes, inner = rng.choice([(96, 64), (8, 32), (48, 128), (7, 33)])
        case = reorder("", dtype, size(1, max(1, 32 * 96 * 2048 * 64 // (width * planes * capacity * inner) if capacity > 256 else 8)),
                       width, planes, capacity, size(1, capacity), inner)
    else:
        capacity = size(16, 4096)
        case = reorder("", rng.choice(["int64", "int32"]), size(1, 64), rng.choice([1, 2, 4, 5, 8]), 1, capacity,
                       size(1, capacity), 1)
    del case["name"]
    return case


def widths_of(case):
    return tuple(int(w) for w in case["widths"].split("+"))


def host_rng(case, seed):
    return random.Random("%d %r" % (seed, sorted((k, v) for k, v in case.items() if k != "name")))


def counts_of(case):
    """The rows of each sequence: the case's own, whatever the seed, as they are the outputs' shapes."""
    rng, rows = host_rng(case, 0), case["rows"]
    counts = [rng.randint(max(1, rows // 4), rows) if case["ragged"] else rows for _ in range(case["seqs"])]
    counts[0] = rows
    return counts


# -- what a pass has in hand -----------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device=CUDA).manual_seed(seed)
    return {"lora": prepare_lora, "beams": prepare_beams, "reorder": prepare_reorder}[case["kind"]](case, seed, g)


def put(values, dtype):
    return torch.tensor(values, device=CUDA, dtype=dtype)


def prepare_lora(case, seed, g):
    rng = host_rng(case, seed + 1)
    n, slots, rank, inputs = case["seqs"], case["slots"], case["rank"], case["inputs"]
    widths, dtype, wtype = widths_of(case), TYPES[case["dtype"]], TYPES[case["wtype"]]
    counts = counts_of(case)
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = int(starts[-1])
    # Sequences in the order of their arrival: the adapters of a batch lie anywhere among them and among the slots.
    used = rng.sample(range(slots), case["adapters"])
    ids = used + [rng.choice(used) for _ in range(n - len(used))]
    if case["none"]:
        free = [i for i in range(len(used), n)]
        for i in free[: n // case["none"]]:
            ids[i] = -1
    rng.shuffle(ids)
    ranks = [max(1, rank >> rng.randrange(4)) if case["mixed_ranks"] else rank for _ in range(slots)]
    a = torch.randn(slots, len(widths) * rank, inputs, device=CUDA, generator=g) * inputs ** -0.5
    b = torch.randn(slots, sum(widths), rank, device=CUDA, generator=g) * 0.1
    x = torch.randn(rows, inputs, device=CUDA, generator=g)
    x = x * (1 + 9 * (torch.rand(inputs, device=CUDA, generator=g) < 0.01))             # a few channels stand out
    base = torch.randn(rows, sum(widths), device=CUDA, generator=g) * 2
    state = {"case": case, "a": a.to(wtype), "b": b.to(wtype), "x": x.to(dtype), "base": base.to(dtype),
             "out": torch.empty(rows, sum(widths), device=CUDA, dtype=dtype),
             "adapters": put(ids, torch.int32), "row_start": put(starts, torch.int32),
             "ranks": put(ranks, torch.int32), "scales": put([2.0 * 16 / r for r in ranks], torch.float32),
             "host": (ids, counts, ranks)}
    # A program that multiplies an adapter at a time keeps its rows at hand.
    where = {}
    for i, s in enumerate(ids):
        if s >= 0:
            where.setdefault(s, []).extend(range(starts[i], starts[i + 1]))
    state["where"] = {s: put(r, torch.int64) for s, r in where.items()}
    if own:
        from nanocompile_b200 import serving

        state["layout"] = serving.LoraLayout(inputs, widths, rank)
        state["batch"] = batch = serving.LoraBatch(rows, n, slots)
        state["plan"] = torch.zeros(batch.plan_bytes, device=CUDA, dtype=torch.uint8)
        serving.lora_plan(batch, state["plan"], state["adapters"], row_start=state["row_start"], stream=stream())
    return state


def prepare_beams(case, seed, g):
    groups, width, vocab = case["groups"], case["beams"], case["vocab"]
    rows = groups * width
    # Logits as a language model gives them: a broad bulk and a few tokens well above it.
    logits = torch.randn(rows, vocab, device=CUDA, generator=g) * 2.0
    peaks = torch.randint(0, vocab, (rows, min(8, vocab)), device=CUDA, generator=g)
    logits.scatter_add_(1, peaks, torch.rand(peaks.shape, device=CUDA, generator=g) * 12)
    if case["masked"]:                                         # a constrained step: part of the vocabulary is out
        logits[:, torch.rand(vocab, device=CUDA, generator=g) < 0.25] = -math.inf
    # Beams of a request lie close to one another; one in sixteen is not there (yet), one in eight has ended.
    scores = torch.randn(rows, device=CUDA, generator=g) * 1.5 - 20 * torch.rand(groups, 1, device=CUDA, generator=g).expand(-1, width).reshape(-1) - 5
    gone = torch.rand(rows, device=CUDA, generator=g) < 1 / 16
    gone[::width] = False
    ended = (torch.rand(rows, device=CUDA, generator=g) < 1 / 8) & bool(case["finished"])
    state = {"case": case, "logits": logits.to(TYPES[case["dtype"]]), "scores": torch.where(gone, -math.inf, scores),
             "finished": ended.to(torch.int32), "end": min(7, vocab - 1),
             "norms": torch.rand(rows, device=CUDA, generator=g) * 3 + 4 if case["norms"] else None}
    for name, dtype in (("parent", torch.int32), ("tokens", torch.int64), ("new_scores", torch.float32),
                        ("new_finished", torch.int32), ("grow", torch.int32), ("history", torch.int32)):
        state[name] = torch.empty(rows, device=CUDA, dtype=dtype)
    if own:
        from nanocompile_b200 import serving

        state["scratch"] = torch.zeros(serving.beam_select_scratch_bytes(rows, vocab, width), device=CUDA, dtype=torch.uint8)
    return state


def prepare_reorder(case, seed, g):
    rng = host_rng(case, seed)
    rows, width, capacity = case["groups"] * case["beams"], case["beams"], case["capacity"]
    shape = (rows, case["planes"], capacity, case["inner"])
    if case["dtype"].startswith("int"):
        dtype = getattr(torch, case["dtype"])
        old, new = (torch.randint(0, 151936, shape, device=CUDA, generator=g, dtype=dtype) for _ in range(2))
        more = torch.randint(0, 151936, (rows, case["planes"], case["inner"]), device=CUDA, generator=g, dtype=dtype)
    else:
        dtype = TYPES[case["dtype"]]
        old = torch.randn(shape, device=CUDA, generator=g).to(dtype)
        new = torch.zeros(shape, device=CUDA, dtype=dtype)
        more = torch.randn(rows, case["planes"], case["inner"], device=CUDA, generator=g).to(dtype)
    lengths = [case["length"] if f == 0 else rng.randint((case["length"] + 1) // 2, case["length"]) for f in range(case["groups"])]
    lengths = [m for m in lengths for _ in range(width)]
    parent = [i - i % width + rng.randrange(width) for i in range(rows)]
    if rows > 8:
        parent[rows // 2] = -1                                                       # a beam that has ended and gone
    return {"case": case, "old": old, "new": new, "append": more, "parent": put(parent, torch.int32),
            "lengths": put(lengths, torch.int32), "new_lengths": torch.zeros(rows, device=CUDA, dtype=torch.int32)}


# -- one pass ------------------------------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"lora": own_lora, "beams": own_beams, "reorder": own_reorder}[kind](state)
    return {"lora": plain_lora, "beams": plain_beams, "reorder": plain_reorder}[kind](state)


def stream():
    return torch.cuda.current_stream().cuda_stream


def own_lora(state):
    from nanocompile_b200 import serving

    at = stream()
    if state["case"]["fresh"]:
        serving.lora_plan(state["batch"], state["plan"], state["adapters"], row_start=state["row_start"], stream=at)
    serving.lora_project(state["layout"], state["batch"], state["out"], state["x"], state["a"], state["b"], state["plan"],
                         base=state["base"], ranks=state["ranks"], scales=state["scales"], stream=at)
    return state["out"]


def own_beams(state):
    from nanocompile_b200 import serving

    serving.beam_select(state["parent"], state["tokens"], state["new_scores"], state["logits"], state["scores"], state["scratch"],
                        beams=state["case"]["beams"], end=state["end"], finished=state["finished"],
                        new_finished=state["new_finished"], grow=state["grow"], history=state["history"], norms=state["norms"],
                        stream=stream())
    return tuple(state[k] for k in ("parent", "tokens", "new_scores", "new_finished", "grow", "history"))


def own_reorder(state):
    from nanocompile_b200 import serving

    serving.beam_reorder(state["new"], state["old"], state["parent"], lengths=state["lengths"], new_lengths=state["new_lengths"],
                         append=state["append"], stream=stream())
    return state["new"], state["new_lengths"]


# -- the plain forms -------------------------------------------------------------------------------------------


def plain_lora(state):
    """An adapter at a time, its rows gathered; everything in 32 bits."""
    case, widths = state["case"], widths_of(state["case"])
    rank, ranks = case["rank"], state["host"][2]
    out = state["base"].to(torch.float32, copy=True)
    for s, rows in state["where"].items():
        x, r = state["x"][rows].float(), ranks[s]
        parts, at = [], 0
        for t, w in enumerate(widths):
            h = x @ state["a"][s, t * rank: t * rank + r].float().T
            parts.append(h @ state["b"][s, at: at + w, :r].float().T)
            at += w
        out[rows] += torch.cat(parts, 1) * state["scales"][s]
    return out.to(state["x"].dtype)


def plain_beams(state):
    """The best `beams` of each row, then those of each request; sums in 64 bits, as totals may lie close together."""
    case = state["case"]
    groups, width, vocab, end = case["groups"], case["beams"], case["vocab"], state["end"]
    x = state["logits"].float()
    live = (state["finished"] == 0) & (state["scores"] > -math.inf)
    top = x.amax(-1, keepdim=True)
    centred = x - torch.where(top > -math.inf, top, 0.0)
    log_sum = top[:, 0].double() + torch.log(torch.exp(centred).sum(-1, dtype=torch.float64))
    # The largest logits, the lowest index first among equals: one whole number orders both.
    bits = x.view(torch.int32).long() & 0xFFFFFFFF
    bits = torch.where(x == 0, 0, bits)
    order = torch.where(bits >= 2**31, 2**32 - 1 - bits, bits + 2**31) - 2**31
    k = min(width, vocab)
    key = order * 2**32 + (2**32 - 1 - torch.arange(vocab, device=CUDA))
    ids = 2**32 - 1 - (torch.topk(key, k, dim=-1).values & 0xFFFFFFFF)
    best = x.gather(1, ids).double()
    scores = state["scores"].double()
    total = torch.where(live[:, None] & (best > -math.inf), scores[:, None] + (best - log_sum[:, None]), -math.inf)
    ended = (state["finished"] != 0) & (scores > -math.inf)
    total[:, 0] = torch.where(ended, scores, total[:, 0])
    ids = torch.where(ended[:, None], end, ids)
    by = total if state["norms"] is None else total / state["norms"].double()[:, None]
    by, total, ids = (v.view(groups, width * k) for v in (by, total, ids))
    chosen = torch.sort(by, dim=-1, descending=True, stable=True).indices
    chosen = chosen[:, :width]
    if chosen.shape[1] < width:
        raise ValueError("fewer candidates than beams")
    picked = total.gather(1, chosen).flatten()
    there = picked > -math.inf
    parent = (torch.arange(groups, device=CUDA)[:, None] * width + chosen // k).flatten()
    tokens = ids.gather(1, chosen).flatten()
    was = ended[parent]
    done = there & (was | (tokens == end))
    return (torch.where(there, parent, -1).to(torch.int32), torch.where(there, tokens, end),
            torch.where(there, picked, -math.inf).float(), (done | ~there).to(torch.int32),
            (there & ~was).to(torch.int32), torch.where(there & ~done, parent, -1).to(torch.int32))


def plain_reorder(state):
    capacity, old, new = state["case"]["capacity"], state["old"], state["new"]
    parent = state["parent"].long()
    there = parent >= 0
    source = parent.clamp(min=0)
    lengths = torch.where(there, state["lengths"][source].long(), -1)
    at = torch.arange(capacity, device=CUDA)
    kept = (at < lengths[:, None])[:, None, :, None]
    moved = torch.where(kept, old[source], new)
    last = (at == lengths[:, None])[:, None, :, None]
    new.copy_(torch.where(last, state["append"][:, :, None], moved))
    return new, torch.where(there, (lengths + 1).clamp(max=capacity), 0).to(torch.int32)


# -- what a pass cannot do without -----------------------------------------------------------------------------


def work(case):
    if case["kind"] == "lora":
        size = 4 if case["dtype"] == "float32" else 2
        n, outputs, targets = case["seqs"], sum(widths_of(case)), len(widths_of(case))
        rows = case["rows"] * (1 + (n - 1) * (0.625 if case["ragged"] else 1))
        rank = case["rank"] * (0.46875 if case["mixed_ranks"] else 1)
        without = min(n // case["none"], n - case["adapters"]) / n if case["none"] else 0
        weights = case["adapters"] * rank * (targets * case["inputs"] + outputs) * 2
        return {"bytes": int(weights + rows * ((1 - without) * case["inputs"] + 2 * outputs) * size + 8 * n),
                "flops": int(2 * rows * (1 - without) * rank * (targets * case["inputs"] + outputs))}
    if case["kind"] == "beams":
        size = 4 if case["dtype"] == "float32" else 2
        rows = case["groups"] * case["beams"]
        live = (rows - case["groups"]) * 15 / 16 + case["groups"]
        live *= 7 / 8 if case["finished"] else 1
        return {"bytes": int(live * case["vocab"] * size + rows * (12 + 28)), "flops": int(4 * live * case["vocab"])}
    size = {"float32": 4, "int32": 4, "int64": 8}.get(case["dtype"], 2)
    groups, width = case["groups"], case["beams"]
    positions = case["length"] * (1 + 0.75 * (groups - 1)) * width
    line = case["planes"] * case["inner"] * size
    return {"bytes": int(2 * (positions + groups * width) * line), "flops": 0}


# -- the definition, in 64 bits ----------------------------------------------------------------------------------


def exact(case, seed):
    if case["kind"] == "reorder":
        return None
    state = prepare(case, seed)
    return exact_lora(case, state) if case["kind"] == "lora" else exact_beams(case, state)


def exact_lora(case, state):
    """A sequence at a time."""
    ids, counts, ranks = state["host"]
    widths, rank = widths_of(case), case["rank"]
    out, at = state["base"].double(), 0
    for s, count in zip(ids, counts):
        rows = slice(at, at + count)
        at += count
        if s < 0:
            continue
        low = torch.einsum("rk,jk->rj", state["x"][rows].double(), state["a"][s].double())
        n = 0
        for t, w in enumerate(widths):
            h = low[:, t * rank: t * rank + ranks[s]]
            delta = torch.einsum("rj,nj->rn", h, state["b"][s, n: n + w, : ranks[s]].double())
            out[rows, n: n + w] += delta * float(state["scales"][s])
            n += w
    return out


def exact_beams(case, state):
    """A request at a time: all candidates of all its beams in one order."""
    groups, width, vocab, end = case["groups"], case["beams"], case["vocab"], state["end"]
    out = []
    for g in range(groups):
        rows = range(g * width, (g + 1) * width)
        x = state["logits"][g * width: (g + 1) * width].double()
        s = state["scores"][g * width: (g + 1) * width].double()
        f = state["finished"][g * width: (g + 1) * width] != 0
        total = s[:, None] + torch.log_softmax(x, -1)
        itself = torch.full_like(total, -math.inf)
        itself[:, end] = s
        total = torch.where(f[:, None], itself, total)
        by = total if state["norms"] is None else total / state["norms"][g * width: (g + 1) * width].double()[:, None]
        order = torch.sort(by.flatten(), descending=True, stable=True).indices[:width]
        best = total.flatten()[order]
        beam, token = order // vocab, order % vocab
        there = best > -math.inf
        done = there & (f[beam] | (token == end))
        row = rows[0] + beam
        out.append((torch.where(there, row, -1).int(), torch.where(there, token, end), best, (done | ~there).int(),
                    (there & ~f[beam]).int(), torch.where(there & ~done, row, -1).int()))
    return tuple(torch.cat(parts) for parts in zip(*out))
