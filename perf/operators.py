"""What is measured of the operators of the int8 key/value cache: writing it
(RoPE, quantising, append), reading rows back, attention of single tokens over
it and attention of many rows over it, both with an optional sliding window
and first tokens that stay visible.

A cache holds int8 planes k and v [slot][kv head][context][head_dim] and fp32
scales [slot][kv head][block of tokens]; an element stands for q * scale.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
TINY = 2.0 ** -126


# ------------------------------------------------------------------- cases

def listed():
    small = {"heads": 9, "kv_heads": 3, "head_dim": 64, "context": 2048, "block": 64}  # the SmolLM2-135M layout
    wide = {"heads": 32, "kv_heads": 8, "head_dim": 128}
    return [
        # One new token for each of 32 sequences between 512 and 2047 tokens: a layer of a decode step.
        {"name": "append-step", "op": "append", **small, "batch": 32, "low": 1, "high": 1, "past": 2046},
        # 32 prompts of 512 tokens written at once.
        {"name": "append-prompts", "op": "append", **small, "batch": 32, "low": 512, "high": 512, "past": 0},
        # Chunks of prompts of odd lengths, most of them begun inside a block.
        {"name": "append-ragged", "op": "append", **wide, "context": 4096, "block": 32, "batch": 13, "low": 1,
         "high": 1531, "past": 2500},
        # A look at one short sequence.
        {"name": "read-short", "op": "read", **small, "batch": 1, "low": 77, "high": 77, "past": 13},
        # Whole sequences of a batch handed to a path that wants fp32.
        {"name": "read-batch", "op": "read", **wide, "context": 2048, "block": 128, "batch": 16, "low": 900,
         "high": 1777, "past": 200},
        # The first tokens of one sequence: only latency counts.
        {"name": "decode-one", "op": "decode", **small, "batch": 1, "low": 37, "high": 37, "window": 0, "sinks": 0},
        # A decode step of 32 sequences from 512 to 2048 tokens, two of them finished.
        {"name": "decode-batch", "op": "decode", **small, "batch": 32, "low": 512, "high": 2048, "window": 0,
         "sinks": 0, "finished": 2},
        # A few long sequences.
        {"name": "decode-long", "op": "decode", **wide, "context": 65536, "block": 64, "batch": 4, "low": 40001,
         "high": 65536, "window": 0, "sinks": 0},
        # Long streams of which each token sees the last 1024 and the first 4.
        {"name": "decode-window", "op": "decode", "heads": 16, "kv_heads": 2, "head_dim": 64, "context": 16384,
         "block": 32, "batch": 24, "low": 2000, "high": 16384, "window": 1024, "sinks": 4},
        # Five drafted tokens for each of 32 sequences, scored at once.
        {"name": "prefill-drafts", "op": "prefill", **small, "batch": 32, "low": 5, "high": 5, "past": 1500,
         "window": 0, "sinks": 0},
        # The prompts of a batch.
        {"name": "prefill-prompts", "op": "prefill", **small, "batch": 32, "low": 512, "high": 512, "past": 0,
         "window": 0, "sinks": 0},
        # A chunk of a long prompt, with a window.
        {"name": "prefill-long", "op": "prefill", **wide, "context": 16384, "block": 64, "batch": 2, "low": 1500,
         "high": 2047, "past": 14000, "window": 4096, "sinks": 16},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "read", "decode", "decode", "prefill", "prefill"])
    head_dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
    case = {"op": op, "heads": kv_heads * group, "kv_heads": kv_heads, "head_dim": head_dim,
            "block": rng.choice([32, 64, 128])}
    if op == "decode":
        batch = log(1, 48)
        high = log(1, min(65536, 262144 * 8 // (batch * kv_heads)))
        window = rng.choice([0, 0, log(1, high)])
        case |= {"batch": batch, "low": max(1, high // rng.choice([1, 2, 5])), "high": high,
                 "context": high + log(1, 64) - 1, "window": window,
                 "sinks": rng.choice([0, 1, 4, 33]) if window else 0}
        return case
    batch = log(1, 32)
    high = log(1, max(1, min(4096, 81920 // case["heads"]) // batch))
    past = rng.choice([0, log(1, 4000), log(1, 400)])
    case |= {"batch": batch, "low": max(1, high // rng.choice([1, 2, 7])), "high": high, "past": past,
             "context": high + past + log(1, 64) - 1}
    if op == "prefill":
        window = rng.choice([0, 0, log(1, high + past)])
        case |= {"window": window, "sinks": rng.choice([0, 1, 4, 33]) if window else 0}
    return case


def _lengths(case, seed):
    """Rows of each sequence (decode: its tokens), and the tokens before them: the case's own set, in an order that
    goes by the seed."""
    rng = np.random.default_rng([case["batch"], case["low"], case["high"], case["context"]])
    n, low, high = case["batch"], case["low"], case["high"]
    count = rng.integers(low, high + 1, n)
    count[0] = high
    past = np.zeros(n, np.int64)
    if case["op"] != "decode":
        past = np.minimum(rng.integers(case["past"] // 4, case["past"] + 1, n), case["context"] - count)
    order = np.random.default_rng(seed).permutation(n)
    return count[order], past[order]


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    h, kv, d, ctx, block = (case[x] for x in ("heads", "kv_heads", "head_dim", "context", "block"))
    n = case["batch"]
    count, past = _lengths(case, seed)
    state = {"case": case, "block": block, "heads": h}

    def ints(a):
        return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    # A cache in use: integers spread over the range of their blocks, scales of nearby powers of two.
    for name, exponent in (("k", -5), ("v", -6)):
        plane = torch.empty(n, kv, ctx, d, dtype=torch.int8, device=DEV)
        for s in range(n):
            plane[s] = (randn(kv, ctx, d) * 40).round_().clamp_(-127, 127).to(torch.int8)
        state[name] = plane
        e = torch.randint(-1, 2, (n, kv, -(-ctx // block)), generator=g, device=DEV)
        state[name + "_scale"] = torch.exp2(e.float() + exponent)

    if case["op"] == "decode":
        pos = count - 1
        for i in range(case.get("finished", 0)):
            pos[1 + 3 * i] = -1
        state["row_pos"] = ints(pos)
        state["q"] = randn(n, h * d) * 0.8
        state["out"] = torch.zeros(n, h * d, device=DEV)
        return state

    rows = int(count.sum())
    state |= {"first": ints(np.cumsum(count) - count), "count": ints(count), "pos0": ints(past), "rows": rows,
              "max_rows": int(count.max())}
    if case["op"] == "prefill":
        state["q"] = randn(rows, h * d) * 0.8
        state["out"] = torch.zeros(rows, h * d, device=DEV)
        return state
    if case["op"] == "append":
        # Keys have a few channels that are larger throughout, and some tokens are larger than others.
        x = randn(rows, (h + 2 * kv) * d)
        x *= torch.exp2(torch.randint(-1, 2, (rows, 1), generator=g, device=DEV).float())
        x[:, h * d:(h + kv) * d] *= torch.exp(0.6 * randn(kv * d))
        state["qkv"] = x
        state["q_out"] = torch.zeros(rows, h * d, device=DEV)
        angle = np.outer(np.arange(ctx), 10000.0 ** (-np.arange(0, d, 2) / d))
        angle = np.concatenate([angle, angle], axis=1)
        state["cos"] = torch.tensor(np.cos(angle), dtype=torch.float32, device=DEV)
        state["sin"] = torch.tensor(np.sin(angle), dtype=torch.float32, device=DEV)
        # What is read back: the blocks that the rows went to, from their first token.
        start = past // block * block
    else:
        start = past
    back = past + count - start
    state |= {"back_first": ints(np.cumsum(back) - back), "back_count": ints(back), "back_pos0": ints(start),
              "back_rows": int(back.sum()), "back_max": int(back.max())}
    state["k_out"] = torch.zeros(int(back.sum()), kv * d, device=DEV)
    state["v_out"] = torch.zeros(int(back.sum()), kv * d, device=DEV)
    return state


# --------------------------------------------------------------- the passes

def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    if op == "append":
        _plain_append(state)
        out = _plain_read(state)
        out["q"] = state["q_out"]
        return out
    if op == "read":
        return _plain_read(state)
    if op == "decode":
        return _plain_decode(state)
    return _plain_prefill(state)


def _own(state, op):
    from accelep_b200 import kernels as K

    s = state
    if "cache" not in s:  # the handle and the workspace that a serving loop keeps
        s["cache"] = K.Q8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"], s["block"])
        if op == "decode":
            s["workspace"] = K.attention_decode_q8_workspace(s["cache"], s["q"].shape[0], s["heads"],
                                                             s["case"]["window"], s["case"]["sinks"])
        if op == "prefill":
            s["workspace"] = K.attention_prefill_q8_workspace(s["cache"], s["count"].shape[0], s["max_rows"],
                                                              s["heads"], s["case"]["window"], s["case"]["sinks"])
    cache = s["cache"]
    if op == "decode":
        return K.attention_decode_q8(s["q"], cache, s["row_pos"], s["heads"], window=s["case"]["window"],
                                     sinks=s["case"]["sinks"], out=s["out"], workspace=s["workspace"])
    if op == "prefill":
        return K.attention_prefill_q8(s["q"], cache, s["first"], s["count"], s["pos0"], s["heads"], s["max_rows"],
                                      window=s["case"]["window"], sinks=s["case"]["sinks"], out=s["out"],
                                      workspace=s["workspace"])
    if op == "append":
        K.rope_append_q8(s["qkv"], cache, s["first"], s["count"], s["pos0"], s["heads"], s["max_rows"], s["cos"],
                         s["sin"], q_out=s["q_out"])
    K.cache_rows_q8(cache, s["back_first"], s["back_count"], s["back_pos0"], s["back_max"], s["k_out"], s["v_out"])
    out = {"k": s["k_out"], "v": s["v_out"]}
    return {**out, "q": s["q_out"]} if op == "append" else out


def _rows(first, count, pos0, rows):
    """The sequence and the position of each of `rows` rows."""
    seq = torch.repeat_interleave(torch.arange(count.shape[0], device=count.device), count.long(), output_size=rows)
    return seq, pos0.long()[seq] + torch.arange(rows, device=count.device) - first.long()[seq]


def _dequantised(plane, scale, block):
    each = scale.repeat_interleave(block, dim=2)[:, :, :plane.shape[2]]
    return plane.float() * each.unsqueeze(-1)


def _rotated(x, cos, sin):
    """Rotate-half RoPE of x [rows, heads, d] with rows of cos and sin [rows, d]."""
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    cos, sin = cos.unsqueeze(1), sin.unsqueeze(1)
    return torch.cat([a * cos[..., :half] - b * sin[..., :half], b * cos[..., half:] + a * sin[..., half:]], dim=-1)


def _power(amax):
    """The least power of two s (2^-126 at least) with amax <= 127 * s."""
    m, e = torch.frexp(amax)
    e = torch.where(m <= 127.0 / 128.0, e - 7, e - 6)
    e = torch.where(amax > 0, e, -126).clamp_(min=-126)
    return ((e + 127) << 23).view(torch.float32)


def _plain_append(state):
    h, kv, d, block = (state["case"][x] for x in ("heads", "kv_heads", "head_dim", "block"))
    seq, pos = _rows(state["first"], state["count"], state["pos0"], state["rows"])
    x = state["qkv"].view(state["rows"], h + 2 * kv, d)
    cos, sin = state["cos"][pos], state["sin"][pos]
    state["q_out"].copy_(_rotated(x[:, :h], cos, sin).flatten(1))
    pos0 = state["pos0"].long()
    slot = torch.arange(pos0.shape[0], device=pos0.device)
    old = pos0 % block  # tokens that the first block of each sequence already holds
    first_block = (pos0 // block).clamp(max=state["k_scale"].shape[2] - 1)
    for name, new in (("k", _rotated(x[:, h:h + kv], cos, sin)), ("v", x[:, h + kv:])):
        plane, scale = state[name], state[name + "_scale"]
        blocks = scale.shape[2]
        amax = torch.zeros(scale.shape[0] * blocks, kv, device=x.device)
        amax.index_reduce_(0, seq * blocks + pos // block, new.abs().amax(-1), "amax")
        amax = amax.view(-1, blocks, kv).transpose(1, 2)
        touched = torch.zeros(scale.shape[0], blocks, dtype=torch.bool, device=x.device)
        touched[seq, pos // block] = True
        held = torch.zeros_like(touched)
        held[slot, first_block] = old > 0
        keep = held.unsqueeze(1) & (scale * 127 >= amax)
        now = torch.where(touched.unsqueeze(1) & ~keep, _power(amax), scale)
        # The rows that the first block held, at its new scale.
        ratio = torch.gather(scale / now, 2, first_block.view(-1, 1, 1).expand(-1, kv, 1))
        t = torch.arange(block, device=x.device)
        at = (first_block.unsqueeze(1) * block + t).clamp(max=plane.shape[2] - 1)
        rows = plane[slot.unsqueeze(1), :, at]  # [slot, block, kv, d]
        again = torch.round(rows.float() * ratio.view(-1, 1, kv, 1)).clamp(-127, 127).to(torch.int8)
        where = (t < old.unsqueeze(1)).nonzero(as_tuple=True)
        plane[where[0], :, at[where]] = again[where]
        scale.copy_(now)
        plane[seq, :, pos] = torch.round(new / scale[seq, :, pos // block].unsqueeze(-1)).clamp(-127, 127).to(torch.int8)


def _plain_read(state):
    seq, pos = _rows(state["back_first"], state["back_count"], state["back_pos0"], state["back_rows"])
    out = {}
    for name in ("k", "v"):
        scale = state[name + "_scale"][seq, :, pos // state["block"]]
        out[name] = (state[name][seq, :, pos].float() * scale.unsqueeze(-1)).flatten(1)
    return out


def _visible(pos, length, window, sinks):
    """[..., length]: whether the row at position pos sees each token."""
    t = torch.arange(length, device=pos.device)
    pos = pos.unsqueeze(-1)
    near = t > pos - window if window else torch.ones_like(t, dtype=torch.bool)
    return (t <= pos) & (near | (t < sinks))


def _attended(q, k, v, mask):
    """q [n, kv, rows, d], k and v [n, kv, length, d], mask [n, 1, rows, length]."""
    s = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(q.shape[-1]))
    s = torch.where(mask, s, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    return torch.matmul(p, v) / p.sum(-1, keepdim=True)


def _plain_decode(state):
    c = state["case"]
    n, kv, d, g = c["batch"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    pos, length = state["row_pos"].long(), c["high"]
    k = _dequantised(state["k"][:, :, :length], state["k_scale"], c["block"])
    v = _dequantised(state["v"][:, :, :length], state["v_scale"], c["block"])
    mask = _visible(pos.clamp(min=0), length, c["window"], c["sinks"]).view(n, 1, 1, length)
    out = _attended(state["q"].view(n, kv, g, d), k, v, mask).reshape(n, -1)
    return torch.where((pos >= 0).unsqueeze(1), out, state["out"])


def _plain_prefill(state):
    c = state["case"]
    n, kv, d, g = c["batch"], c["kv_heads"], c["head_dim"], c["heads"] // c["kv_heads"]
    rows, m, length = state["rows"], state["max_rows"], c["high"] + c["past"]
    length = min(length, c["context"])
    seq, pos = _rows(state["first"], state["count"], state["pos0"], rows)
    at = pos - state["pos0"].long()[seq]
    q = torch.zeros(n, m, kv * g * d, device=DEV)
    q[seq, at] = state["q"]
    q = q.view(n, m, kv, g, d).permute(0, 2, 1, 3, 4).reshape(n, kv, m * g, d)
    k = _dequantised(state["k"][:, :, :length], state["k_scale"], c["block"])
    v = _dequantised(state["v"][:, :, :length], state["v_scale"], c["block"])
    every = state["pos0"].long().unsqueeze(1) + torch.arange(m, device=DEV)
    mask = _visible(every, length, c["window"], c["sinks"])
    mask = mask.repeat_interleave(g, dim=1).unsqueeze(1)
    # Rows behind the end of a sequence are not used; they see the first token so that their sums are not zero.
    mask = mask | (torch.arange(length, device=DEV) == 0) & (every >= length).repeat_interleave(g, dim=1).view(n, 1, -1, 1)
    out = _attended(q, k, v, mask).view(n, kv, m, g, d).permute(0, 2, 1, 3, 4).reshape(n, m, -1)
    return out[seq, at]


# ------------------------------------------------------------ what it takes

def _seen(case, pos):
    """Tokens that the row at each position sees."""
    pos = np.asarray(pos, np.int64)
    if not case["window"]:
        return pos + 1
    near = np.minimum(pos + 1, case["window"])
    return near + np.minimum(case["sinks"], pos + 1 - near)


def work(case):
    h, kv, d, block = (case[x] for x in ("heads", "kv_heads", "head_dim", "block"))
    # Lengths differ from seed to seed: their mean.
    n, mean = case["batch"], (case["low"] + case["high"]) / 2
    if case["op"] == "decode":
        n = n - case.get("finished", 0)
        pos = np.linspace(case["low"], case["high"], 64).astype(np.int64) - 1
        seen = float(_seen(case, pos).mean())
        return {"bytes": int(n * (2 * kv * (seen * d + 4 * seen / block) + 8 * h * d)), "flops": int(n * 4 * h * d * seen)}
    rows, past = n * mean, case["past"] * 0.625
    back = n * (mean + (min(past, block / 2) if case["op"] == "append" else 0))
    if case["op"] == "prefill":
        at = np.linspace(0, mean - 1, 64) + past
        seen = float(_seen(case, at.astype(np.int64)).mean())
        first = int(_seen(case, int(past)))
        tokens = min(first + mean - 1, mean + past)
        return {"bytes": int(n * 2 * kv * (tokens * d + 4 * tokens / block) + 8 * rows * h * d),
                "flops": int(4 * h * d * rows * seen)}
    read = 2 * kv * (back * 5 * d + 4 * back / block)
    if case["op"] == "read":
        return {"bytes": int(read), "flops": int(2 * kv * back * d)}
    write = rows * d * (4 * (h + 2 * kv) + 4 * h + 2 * kv) + 8 * d * mean + 8 * kv * rows / block
    return {"bytes": int(write + read), "flops": int(rows * d * (3 * (h + kv) + 4 * kv) + 2 * kv * back * d)}


# ------------------------------------------------------------- in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op in ("append", "read"):
        return _exact_cache(state, case, op)
    h, kv, d, block = (case[x] for x in ("heads", "kv_heads", "head_dim", "block"))
    g = h // kv
    if op == "decode":
        first, count, pos0 = list(range(case["batch"])), [1] * case["batch"], state["row_pos"].tolist()
    else:
        first, count, pos0 = state["first"].tolist(), state["count"].tolist(), state["pos0"].tolist()
    out = torch.zeros(state["q"].shape[0], h, d, dtype=torch.float64, device=DEV)
    q = state["q"].double().view(-1, h, d)
    for b, (f, c, p0) in enumerate(zip(first, count, pos0)):
        if p0 < 0:
            continue
        length = p0 + c
        t = torch.arange(length, device=DEV)
        for j in range(kv):
            k = state["k"][b, j, :length].double() * state["k_scale"][b, j, t // block].double().unsqueeze(1)
            v = state["v"][b, j, :length].double() * state["v_scale"][b, j, t // block].double().unsqueeze(1)
            for r0 in range(0, c, 512):
                r1 = min(c, r0 + 512)
                p = torch.arange(p0 + r0, p0 + r1, device=DEV).unsqueeze(1)
                hidden = t > p
                if case["window"]:
                    hidden |= (t <= p - case["window"]) & (t >= case["sinks"])
                s = torch.einsum("rgd,td->rgt", q[f + r0:f + r1, j * g:(j + 1) * g], k) / math.sqrt(d)
                s.masked_fill_(hidden.unsqueeze(1), -math.inf)
                out[f + r0:f + r1, j * g:(j + 1) * g] = torch.softmax(s, dim=-1) @ v
    return out.flatten(1)


def _exact_cache(state, case, op):
    h, kv, d, block = (case[x] for x in ("heads", "kv_heads", "head_dim", "block"))

    def f32(x):  # one rounding to 32 bits: RoPE's definition rounds each of its steps
        return x.float().double()

    first, count, pos0 = (state[x].tolist() for x in ("first", "count", "pos0"))
    value = {}
    for name in ("k", "v"):
        each = state[name + "_scale"].double().repeat_interleave(block, dim=2)[:, :, :case["context"], None]
        value[name] = (state[name].double(), each.clone())
    q_out = None
    if op == "append":
        q_out = torch.empty(state["rows"], h, d, dtype=torch.float64, device=DEV)
        half = d // 2
        for b, (f, c, p0) in enumerate(zip(first, count, pos0)):
            x = state["qkv"][f:f + c].double().view(c, h + 2 * kv, d)
            cos = state["cos"][p0:p0 + c].double().unsqueeze(1)
            sin = state["sin"][p0:p0 + c].double().unsqueeze(1)
            r, turned = x[:, :h + kv], torch.cat([-x[:, :h + kv, half:], x[:, :h + kv, :half]], dim=-1)
            q_out[f:f + c] = (r * cos + turned * sin)[:, :h]
            roped = f32(f32(r * cos) + f32(turned * sin))
            for name, new in (("k", roped[:, h:]), ("v", x[:, h + kv:])):
                q, each = value[name]
                for j0 in range(p0 // block * block, p0 + c, block):
                    lo, hi = max(j0, p0), min(j0 + block, p0 + c)
                    part = new[lo - p0:hi - p0].transpose(0, 1)  # [kv, rows, d]
                    amax = part.abs().amax((1, 2)).clamp(min=1e-300)
                    need = torch.exp2(torch.ceil(torch.log2(amax / 127.0))).clamp(min=TINY)
                    need = torch.where(need * 127 < amax, need * 2, need)
                    need = torch.where((need * 63.5 >= amax) & (need > TINY), need / 2, need)
                    if lo > j0:
                        was = each[b, :, j0, 0]
                        need = torch.where(was * 127 >= amax, was, need)
                        q[b, :, j0:lo] = torch.round(q[b, :, j0:lo] * (was / need).view(-1, 1, 1)).clamp(-127, 127)
                    each[b, :, j0:hi] = need.view(-1, 1, 1)
                    q[b, :, lo:hi] = torch.round(part / need.view(-1, 1, 1)).clamp(-127, 127)
    out = {}
    bf, bc, bp = (state[x].tolist() for x in ("back_first", "back_count", "back_pos0"))
    for name in ("k", "v"):
        q, each = value[name]
        rows = torch.empty(state["back_rows"], kv, d, dtype=torch.float64, device=DEV)
        for b, (f, c, p0) in enumerate(zip(bf, bc, bp)):
            rows[f:f + c] = (q[b, :, p0:p0 + c] * each[b, :, p0:p0 + c]).transpose(0, 1)
        out[name] = rows.flatten(1)
    if op == "append":
        out["q"] = q_out.flatten(1)
    return out
