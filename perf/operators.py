"""Operators of quantised and scored generation, as cases to measure: the 4-bit key/value cache (storing rows, reading
them back, one query per sequence attending over it), the log probabilities of given tokens with the entropy and the
likeliest alternatives, and a language-model head whose float32 logits are scored in the same pass.

``run`` computes a case in plain torch operations, or, where ``own`` is set, with the calls a program makes of
``tempo_compiler_b200.ops``. Both read the same inputs.

The 4-bit cache holds, for each sequence and key/value head, tiles of 16 positions; each group of 64 head dimensions is
1152 bytes of a tile: 16 rows of 32 bytes of key codes, 16 rows of value codes (dimension d in byte d / 2, the even one
in the low half), then for each position four bfloat16 words: key scale, key low, value scale, value low. A row of 64
stands for code * scale + low, with low its least value, scale = bfloat16((greatest - least) / 15) and the code
round((x - low) / scale), ties to even, in 0 .. 15 (0 where the scale is 0).
"""

import math

import torch

own = False

GROUP = 64      # dimensions that share a scale
TILE = 16       # positions of a tile
GROUP_BYTES = TILE * (GROUP + 8)


# ---- the cases ----------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decode step of the benchmark's 64-sequence share: a new token of each sequence into its cache
        {"name": "store step 64x12", "op": "store", "seqs": 64, "tokens": 1, "heads": 12, "kv_heads": 12, "head": 64,
         "span": 1151, "padded": 1},
        # ragged prompts of a grouped-query model with 128-wide heads
        {"name": "store prompts 8x1000 gqa", "op": "store", "seqs": 8, "tokens": 1000, "heads": 32, "kv_heads": 8,
         "head": 128, "span": 77, "padded": 0},
        # the prompts of a 64-sequence batch of GPT-2 small, 1024 tokens each
        {"name": "store prompts 64x1024", "op": "store", "seqs": 64, "tokens": 1024, "heads": 12, "kv_heads": 12,
         "head": 64, "span": 0, "padded": 0},
        # single-sequence greedy decode near the end of its 384 positions
        {"name": "attend 1x12 384", "op": "attend", "seqs": 1, "heads": 12, "kv_heads": 12, "head": 64, "low": 384,
         "high": 384},
        # a continuous batch: sequences from one token to a full cache
        {"name": "attend 64x12 ragged", "op": "attend", "seqs": 64, "heads": 12, "kv_heads": 12, "head": 64, "low": 1,
         "high": 1152},
        # the benchmark's 512 sequences after a 1024-token prompt
        {"name": "attend 512x12 1152", "op": "attend", "seqs": 512, "heads": 12, "kv_heads": 12, "head": 64,
         "low": 1025, "high": 1152},
        # two long documents under a grouped-query model
        {"name": "attend 2x32/8 long", "op": "attend", "seqs": 2, "heads": 32, "kv_heads": 8, "head": 128,
         "low": 40001, "high": 65536},
        # one token answered with its five likeliest alternatives
        {"name": "logprobs 1 top5", "op": "logprobs", "rows": 1, "vocab": 50257, "dtype": "float32", "top": 5},
        # a decode step of 512 sequences that reports twenty alternatives
        {"name": "logprobs 512 top20", "op": "logprobs", "rows": 512, "vocab": 50257, "dtype": "float32", "top": 20},
        # the prompt tokens of eight sequences, scored from bfloat16 logits
        {"name": "logprobs 8192 bf16", "op": "logprobs", "rows": 8192, "vocab": 50257, "dtype": "bfloat16", "top": 1},
        # the language-model head and its scores: a small decode batch, and two prompts of 1024 tokens
        {"name": "score 64", "op": "score", "rows": 64, "width": 768, "vocab": 50257},
        {"name": "score 2048", "op": "score", "rows": 2048, "width": 768, "vocab": 50257},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    op = rng.choice(["store", "attend", "logprobs", "score"])
    if op in ("store", "attend"):
        head = rng.choice([64, 128])
        kv_heads = rng.choice([1, 2, 4, 8, 12])
        heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8, 12])
        groups = kv_heads * head // GROUP
        if op == "store":
            rows = _log(rng, 1, 65536 * 12 // groups if groups > 12 else 65536)
            seqs = min(512, _log(rng, 1, rows))
            tokens = max(1, rows // seqs)
            return {"op": op, "seqs": seqs, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head": head,
                    "span": rng.choice([0, 5, _log(rng, 16, 1024)]), "padded": rng.choice([0, 0, 1])}
        seqs = _log(rng, 1, 512)
        high = _log(rng, 1, min(65536, 512 * 12 * 1024 // (seqs * groups)))
        return {"op": op, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "head": head,
                "low": rng.choice([0, 1, high // 2, high]), "high": high}
    if op == "logprobs":
        vocab, dtype = _log(rng, 500, 152064), rng.choice(["float32", "bfloat16"])
        most = 8192 * 50000 // vocab // (2 if dtype == "float32" else 1)
        return {"op": op, "rows": _log(rng, 1, min(8192, most)), "vocab": vocab, "dtype": dtype,
                "top": rng.choice([0, 1, 5, 20, 32])}
    return {"op": op, "rows": _log(rng, 1, 2048), "width": 8 * _log(rng, 8, 128), "vocab": _log(rng, 500, 50257)}


# ---- inputs -------------------------------------------------------------------------------------------------------

def _quantise(x):
    """Codes (0 .. 15, in the rows' own shape), scale and low (bfloat16) of rows of 64."""
    x = x.float()
    low = x.amin(-1, keepdim=True)
    scale = ((x.amax(-1, keepdim=True) - low) / 15).to(torch.bfloat16).float()
    codes = torch.where(scale > 0, torch.round((x - low) / scale).clamp(0, 15), torch.zeros_like(x))
    return codes, scale.to(torch.bfloat16), low.to(torch.bfloat16)


def _rows(shape, generator):
    """Keys or values as a model makes them: unit spread around an offset of each dimension, a few wide rows."""
    x = torch.randn(shape, generator=generator, device="cuda")
    x += 0.5 * torch.randn(shape[-1], generator=generator, device="cuda")
    x *= torch.exp(0.3 * torch.randn((*shape[:-1], 1), generator=generator, device="cuda"))
    return x.to(torch.bfloat16)


def _lengths(case, generator):
    """Cached positions of each sequence: spread evenly from `low` to `high`, in an order drawn from the seed."""
    s = case["seqs"]
    steps = torch.arange(s, device="cuda") * (case["high"] - case["low"]) // max(1, s - 1)
    lengths = case["high"] - steps
    return lengths[torch.randperm(s, generator=generator, device="cuda")].to(torch.int32)


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "store":
        seqs, tokens, heads, kv_heads, head = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "head"))
        start = torch.randint(0, case["span"] + 1, (seqs,), generator=generator, device="cuda")
        capacity = -(-(tokens + case["span"]) // TILE) * TILE
        pos = (start[:, None] + torch.arange(tokens, device="cuda")[None, :]).reshape(-1).to(torch.int32)
        seq = torch.arange(seqs, device="cuda", dtype=torch.int32).repeat_interleave(tokens)
        if case["padded"]:  # the last rows of a padded batch belong to nobody
            pos[-max(1, pos.numel() // 8):] = -1
        qkv = torch.cat([_rows((seqs * tokens, heads, head), generator),
                         _rows((seqs * tokens, kv_heads, head), generator),
                         _rows((seqs * tokens, kv_heads, head), generator)], 1).reshape(seqs * tokens, -1)
        cache = torch.zeros((seqs, kv_heads, capacity // TILE, GROUP_BYTES * head // GROUP), dtype=torch.uint8,
                            device="cuda")
        return {"case": case, "qkv": qkv, "cache": cache, "seq": seq, "pos": pos}
    if op == "attend":
        seqs, heads, kv_heads, head = (case[k] for k in ("seqs", "heads", "kv_heads", "head"))
        tiles, groups = -(-case["high"] // TILE), head // GROUP
        lengths = _lengths(case, generator)
        parts, words = [], []
        for _ in range(2):
            codes, scale, low = _quantise(_rows((seqs, kv_heads, tiles, TILE, groups, GROUP), generator))
            codes = codes.to(torch.uint8).transpose(3, 4).reshape(seqs, kv_heads, tiles, groups, TILE * GROUP)
            parts.append(codes[..., 0::2] | codes[..., 1::2] << 4)
            words += [scale, low]
        words = torch.cat(words, -1).transpose(3, 4).reshape(seqs, kv_heads, tiles, groups, TILE * 4)
        cache = torch.cat([*parts, words.contiguous().view(torch.uint8)], -1)
        q = torch.randn((seqs, heads, head), generator=generator, device="cuda") * (1.5 / math.sqrt(head))
        kv = torch.randn((seqs, 2 * kv_heads, head), generator=generator, device="cuda")
        qkv = torch.cat([q, kv], 1).to(torch.bfloat16).reshape(seqs, -1)
        return {"case": case, "qkv": qkv, "cache": cache.reshape(seqs, kv_heads, tiles, groups * GROUP_BYTES),
                "lengths": lengths}
    rows, vocab = case["rows"], case["vocab"]
    ids = torch.randint(0, vocab, (rows,), generator=generator, device="cuda", dtype=torch.int32)
    if rows > 8:  # a padded batch has rows without a token
        ids[rows - rows // 16 - 1:] = -1
    if op == "logprobs":
        x = torch.randn((rows, vocab), generator=generator, device="cuda")
        x *= 1.0 + 2.0 * torch.rand((rows, 1), generator=generator, device="cuda")
        x -= 30.0
        return {"case": case, "logits": x.to(getattr(torch, case["dtype"])), "ids": ids}
    hidden = torch.randn((rows, case["width"]), generator=generator, device="cuda").to(torch.bfloat16)
    table = (0.1 * torch.randn((vocab, case["width"]), generator=generator, device="cuda")).to(torch.bfloat16)
    # the logits' buffer, whose rows are padded to eight columns, is kept between steps as a program would
    logits = torch.empty((rows, -(-vocab // 8) * 8), dtype=torch.float32, device="cuda")[:, :vocab]
    return {"case": case, "hidden": hidden, "table": table, "logits": logits, "ids": ids}


# ---- one pass -----------------------------------------------------------------------------------------------------

def _split(qkv, case):
    rows, head = qkv.shape[0], case["head"]
    x = qkv.reshape(rows, -1, head)
    return x[:, :case["heads"]], x[:, case["heads"]:]


def _plain_store(state):
    case = state["case"]
    _, kv = _split(state["qkv"], case)
    codes, scale, low = _quantise(kv.reshape(*kv.shape[:2], -1, GROUP))
    value = codes * scale.float() + low.float()
    held = (state["pos"] >= 0)[:, None]
    return torch.where(held, value.reshape(kv.shape[0], -1), torch.zeros((), device="cuda")).to(torch.bfloat16)


def _unpacked(cache, at):
    """Keys (at 0) or values (at 1) of a cache as float32 [seqs, kv_heads, positions, head]."""
    seqs, kv_heads, tiles, size = cache.shape
    groups, codes_bytes = size // GROUP_BYTES, TILE * GROUP // 2
    x = cache.view(seqs, kv_heads, tiles, groups, GROUP_BYTES)
    b = x[..., at * codes_bytes:(at + 1) * codes_bytes].reshape(seqs, kv_heads, tiles, groups, TILE, GROUP // 2)
    words = x[..., 2 * codes_bytes:].contiguous().view(torch.bfloat16).view(seqs, kv_heads, tiles, groups, TILE, 4)
    codes = torch.stack([b & 15, b >> 4], -1).flatten(-2).float()
    value = codes * words[..., 2 * at:2 * at + 1].float() + words[..., 2 * at + 1:2 * at + 2].float()
    return value.transpose(3, 4).reshape(seqs, kv_heads, tiles * TILE, groups * GROUP)


def _plain_attend(state):
    case = state["case"]
    q, _ = _split(state["qkv"], case)
    seqs, kv_heads, head = case["seqs"], case["kv_heads"], case["head"]
    q = q.float().reshape(seqs, kv_heads, -1, head)
    scores = q @ _unpacked(state["cache"], 0).transpose(2, 3)
    held = torch.arange(scores.shape[-1], device="cuda") < state["lengths"][:, None]
    scores = scores.masked_fill(~held[:, None, None, :], -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    out = (e @ _unpacked(state["cache"], 1)) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.reshape(seqs, -1).to(torch.bfloat16)


def _plain_logprobs(logits, ids, top):
    x = logits.float()
    high = x.amax(1, keepdim=True)
    d = x - high.clamp(min=torch.finfo(torch.float32).min)
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    weighted = torch.where(e > 0, d * e, torch.zeros_like(e)).sum(1)
    empty = total == 0
    entropy = torch.where(empty, torch.zeros_like(total), log_total - weighted / total)
    named = (ids >= 0) & (ids < x.shape[1])
    picked = d.gather(1, ids.clamp(0, x.shape[1] - 1).long()[:, None])[:, 0] - log_total
    picked = torch.where(empty, torch.full_like(total, -math.inf), picked)
    logprob = torch.where(named, picked, torch.zeros_like(picked))
    if top == 0:
        return logprob, entropy
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    best = torch.where(empty[:, None], torch.full((1, 1), -math.inf, device="cuda"),
                       d.gather(1, order) - log_total[:, None])
    return logprob, entropy, best, order.to(torch.int32)


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from tempo_compiler_b200 import ops
        if op == "store":
            ops.kv_store_q4(state["qkv"], state["cache"], state["seq"], state["pos"])
            return ops.kv_load_q4(state["cache"], state["seq"], state["pos"])
        if op == "attend":
            return ops.decode_attention_q4(state["qkv"], state["cache"], state["lengths"])
        if op == "logprobs":
            return tuple(ops.token_logprobs(state["logits"], state["ids"], top=case["top"]))
        logits = ops.gemm_f32(state["hidden"], state["table"], out=state["logits"])
        return tuple(ops.token_logprobs(logits, state["ids"]))
    if op == "store":
        return _plain_store(state)
    if op == "attend":
        return _plain_attend(state)
    if op == "logprobs":
        return _plain_logprobs(state["logits"], state["ids"], case["top"])
    return _plain_logprobs(state["hidden"].float() @ state["table"].float().T, state["ids"], 0)


def work(case):
    op = case["op"]
    if op in ("store", "attend"):
        kv = case["kv_heads"] * case["head"]
        held = 2 * kv // 2 + 2 * kv // GROUP * 4  # bytes of one position
        if op == "store":
            rows = case["seqs"] * case["tokens"]
            return {"bytes": rows * (2 * kv * 2 + held + 2 * kv * 2 + 8), "flops": rows * 2 * kv * 6}
        s = case["seqs"]
        total = sum(case["high"] - i * (case["high"] - case["low"]) // max(1, s - 1) for i in range(s))
        q = case["heads"] * case["head"]
        return {"bytes": total * held + s * (4 * q + 4), "flops": 4 * total * q}
    rows, vocab = case["rows"], case["vocab"]
    if op == "logprobs":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": rows * (vocab * size + 12 + 8 * case["top"]), "flops": 5 * rows * vocab}
    width = case["width"]
    return {"bytes": 2 * width * (rows + vocab) + 12 * rows, "flops": 2 * rows * vocab * width}


# ---- the definition, in 64 bits -----------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "store":
        kv = state["qkv"][:, case["heads"] * case["head"]:].double().unflatten(1, (-1, GROUP))
        least, most = kv.min(2).values, kv.max(2).values
        step = ((most - least) / 15).to(torch.bfloat16).double()[..., None]
        least = least[..., None]
        n = torch.nan_to_num((kv - least) / step, nan=0.0, posinf=0.0).round().clamp(0, 15)
        value = (least + n * step).flatten(1)
        value[state["pos"] < 0] = 0
        return value
    if op == "attend":
        return _exact_attend(state)
    if op == "logprobs":
        x = state["logits"]
    else:
        x, table = state["hidden"].double(), state["table"].double()
    parts = []
    block = max(1, 2 ** 26 // case["vocab"])
    for i in range(0, case["rows"], block):
        y = x[i:i + block].double() if op == "logprobs" else x[i:i + block] @ table.T
        parts.append(_exact_logprobs(y, state["ids"][i:i + block], case.get("top", 0)))
    return tuple(torch.cat(p) for p in zip(*parts))


def _exact_attend(state):
    case = state["case"]
    head, groups = case["head"], case["head"] // GROUP
    share = case["heads"] // case["kv_heads"]
    outs = []
    for s in range(case["seqs"]):
        n = int(state["lengths"][s])
        if n == 0:
            outs.append(torch.zeros(case["heads"] * head, dtype=torch.float64, device="cuda"))
            continue
        tiles = state["cache"][s, :, :-(-n // TILE)].unflatten(2, (groups, GROUP_BYTES))
        kv = []
        for offset, word in ((0, 0), (TILE * 32, 2)):
            row = tiles[..., offset:offset + TILE * 32].unflatten(3, (TILE, 32)).long()
            codes = torch.empty((*row.shape[:-1], GROUP), dtype=torch.float64, device="cuda")
            codes[..., 0::2] = (row % 16).double()
            codes[..., 1::2] = (row // 16).double()
            meta = tiles[..., 2 * TILE * 32:].contiguous().view(torch.bfloat16).unflatten(3, (TILE, 4)).double()
            x = codes * meta[..., word, None] + meta[..., word + 1, None]
            kv.append(x.permute(0, 1, 3, 2, 4).flatten(3).flatten(1, 2)[:, :n].repeat_interleave(share, 0))
        q = state["qkv"][s, :case["heads"] * head].double().view(-1, head)
        p = torch.softmax(torch.einsum("hd,hpd->hp", q, kv[0]), 1)
        outs.append(torch.einsum("hp,hpd->hd", p, kv[1]).flatten())
    return torch.stack(outs)


def _exact_logprobs(y, ids, top):
    logs = y - torch.logsumexp(y, 1, keepdim=True)
    inside = (ids >= 0) & (ids < y.shape[1])
    picked = logs[torch.arange(len(ids), device="cuda"), ids.long() * inside] * inside
    entropy = -(logs.exp() * logs).nansum(1)
    if top == 0:
        return picked, entropy
    order = torch.sort(y, dim=1, descending=True, stable=True)[1][:, :top]
    return picked, entropy, logs.gather(1, order), order.int()
