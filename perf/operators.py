"""Performance cases of the serving operators: the key/value cache in pages, the
attention that reads it, and the choice of the next token.

A case is a dict of plain values; its "op" names the operator:

  write      RoPE of a batch's new queries and keys, and the write of its new
             keys and values into the pages, HIPDevice.rope_write_paged
  attention  attention of each sequence's new tokens over its pages, with or
             without a sliding window and first tokens that stay visible,
             HIPDevice.attention_paged
  sample     the next token of each row of logits by temperature, top-k, top-p
             and min-p from given random numbers, HIPDevice.sample

A batch holds `sequences` sequences; sequence s owns rows starts[s] to
starts[s + 1] of the queries, its newest positions, and lengths[s] positions
in all, the new ones among them, on the pages its row of the page table
lists. Heads and widths are those of the repository's Llama shapes (9 over 3
and 32 over 32 heads of 64), and 32 over 8 heads of 128.

With `own` true a pass is the call a program makes; otherwise it is the same
in elementary torch operations, in 32 bits (the sampler's sums in 64).
"""
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16}
THETA = 10000.0


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # One user's decode step, SmolLM2-135M's heads: the smallest write.
        {"name": "write_step", "op": "write", "kind": "F16", "heads": 9, "kv_heads": 3, "width": 64, "page_size": 16,
         "sequences": 1, "new": 1, "longest": 512},
        # Eight users' prompts in one ragged batch, the 1.7B shape's heads.
        {"name": "write_prompts", "op": "write", "kind": "BF16", "heads": 32, "kv_heads": 32, "width": 64,
         "page_size": 32, "sequences": 8, "new": 1024, "longest": 2048},
        # One user's decode step over a short context: the smallest attention, a launch and little else.
        {"name": "decode_1", "op": "attention", "kind": "F16", "heads": 9, "kv_heads": 3, "width": 64,
         "page_size": 16, "sequences": 1, "new": 1, "longest": 512, "window": 0, "sinks": 0},
        # Eight users' decode step, the 1.7B shape, ragged up to its context.
        {"name": "decode_8", "op": "attention", "kind": "BF16", "heads": 32, "kv_heads": 32, "width": 64,
         "page_size": 16, "sequences": 8, "new": 1, "longest": 2048, "window": 0, "sinks": 0},
        # Four users with long documents: a decode step that is all cache reads.
        {"name": "decode_long", "op": "attention", "kind": "F16", "heads": 32, "kv_heads": 8, "width": 128,
         "page_size": 64, "sequences": 4, "new": 1, "longest": 131072, "window": 0, "sinks": 0},
        # Forty-eight endless conversations: a window and the first four tokens, an f32 cache.
        {"name": "decode_window", "op": "attention", "kind": "F32", "heads": 32, "kv_heads": 8, "width": 128,
         "page_size": 16, "sequences": 48, "new": 1, "longest": 8192, "window": 1024, "sinks": 4},
        # A whole prompt of the 1.7B shape's context at once.
        {"name": "prompt", "op": "attention", "kind": "F16", "heads": 32, "kv_heads": 32, "width": 64,
         "page_size": 64, "sequences": 1, "new": 2048, "longest": 2048, "window": 0, "sinks": 0},
        # A later chunk of a long prompt, grouped heads.
        {"name": "chunk", "op": "attention", "kind": "BF16", "heads": 32, "kv_heads": 8, "width": 128,
         "page_size": 32, "sequences": 1, "new": 512, "longest": 30000, "window": 0, "sinks": 0},
        # Chunks and decode steps of twelve users in one batch, odd sizes, window and sinks, an f32 cache.
        {"name": "mixed_window", "op": "attention", "kind": "F32", "heads": 9, "kv_heads": 3, "width": 64,
         "page_size": 24, "sequences": 12, "new": 333, "longest": 1499, "window": 250, "sinks": 3, "mixed": True},
        # One user's next token, SmolLM2's vocabulary, the usual top-k and top-p.
        {"name": "sample_1", "op": "sample", "rows": 1, "n": 49152, "top_k": 40, "top_p": 0.95, "min_p": 0.0,
         "temperature": 0.8, "mixed": False},
        # Thirty-two users of a large vocabulary, top-p alone: long sums.
        {"name": "sample_top_p", "op": "sample", "rows": 32, "n": 131072, "top_k": 0, "top_p": 0.9, "min_p": 0.0,
         "temperature": 1.0, "mixed": False},
        # Two hundred users, each with settings of their own, greedy ones among them.
        {"name": "sample_mixed", "op": "sample", "rows": 200, "n": 50257, "top_k": 100, "top_p": 0.8, "min_p": 0.02,
         "temperature": 1.3, "mixed": True},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["write", "attention", "attention", "attention", "attention", "sample", "sample"])
    if op == "sample":
        n = _log_int(rng, 1000, 150000)
        rows = _log_int(rng, 1, max(1, min(256, 10000000 // n)))
        return {"op": op, "rows": rows, "n": n, "top_k": rng.choice([0, 0, 1, _log_int(rng, 2, 1000)]),
                "top_p": rng.choice([1.0, round(rng.uniform(0.05, 0.99), 3)]),
                "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 4)]),
                "temperature": round(rng.uniform(0.2, 2.0), 2), "mixed": rng.random() < 0.5}
    heads, kv, width = rng.choice([(9, 3, 64), (32, 32, 64), (32, 8, 128), (8, 1, 128), (6, 2, 80), (4, 4, 32),
                                   (10, 5, 256)])
    case = {"op": op, "kind": rng.choice(["F32", "F16", "BF16"]), "heads": heads, "kv_heads": kv, "width": width,
            "page_size": rng.choice([16, 16, 32, 64, 24, 100])}
    if op == "write":
        sequences = _log_int(rng, 1, 64)
        new = rng.choice([1, _log_int(rng, 2, max(2, 8000 // sequences))])
        return dict(case, sequences=sequences, new=new, longest=new + _log_int(rng, 1, 8000))
    what = rng.choice(["decode", "decode", "chunk", "mixed"])
    if what == "decode":
        sequences = _log_int(rng, 1, 64)
        new = rng.choice([1, 1, 1, rng.randint(2, 6)])
        longest = new + _log_int(rng, 16, max(64, min(131072, 800000 // sequences)))
    elif what == "chunk":
        sequences = rng.choice([1, 1, 2, 4])
        new = _log_int(rng, 16, 1024 // sequences)
        longest = new + rng.choice([0, _log_int(rng, 1, 8000)])
    else:
        sequences = rng.randint(3, 24)
        new = _log_int(rng, 8, 400)
        longest = new + _log_int(rng, 1, 4000)
    window = rng.choice([0, 0, _log_int(rng, 16, 4096)])
    return dict(case, sequences=sequences, new=new, longest=longest, window=window,
                sinks=rng.choice([0, 4, rng.randint(1, 64)]) if window else 0, mixed=what == "mixed")


# ------------------------------------------------- inputs, as a program has them

def _batch(case):
    """(new tokens, positions) of each sequence: ragged between a quarter of the case's and the whole of it,
    every third of a mixed batch a decode step."""
    count = case["sequences"]
    part = [0.25 + 0.75 * (s + 1) / count for s in range(count)]
    new = [1 if case.get("mixed") and s % 3 else max(1, round(case["new"] * p)) for s, p in enumerate(part)]
    new[-1] = case["new"]
    return new, [max(n, round(case["longest"] * p)) for n, p in zip(new, part)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * std


def _rope_tables(rows, width):
    freq = 1.0 / torch.pow(torch.tensor(THETA), torch.arange(0, width, 2, dtype=torch.float32) / width)
    angle = torch.arange(rows, dtype=torch.float32)[:, None] * torch.cat([freq, freq])[None]
    return angle.cos().cuda(), angle.sin().cuda()


def _logits(gen, rows, n):
    """What a language model's head gives: most tokens far below a few, by about a logarithm of their rank."""
    rank = torch.rand(rows, n, generator=gen, device="cuda") * n + 1.0
    return _normal(gen, rows, n, std=1.0) - 1.3 * torch.log(rank) + 8.0


def _settings(case, seed):
    """The sampler's settings per row: the case's, or the row's own (a fifth greedy, some steps off)."""
    rows, rng = case["rows"], np.random.default_rng(seed)
    t = np.full(rows, case["temperature"], np.float32)
    k = np.full(rows, case["top_k"], np.int32)
    p = np.full(rows, case["top_p"], np.float32)
    m = np.full(rows, case["min_p"], np.float32)
    if case["mixed"]:
        t *= rng.uniform(0.5, 1.5, rows).astype(np.float32)
        t[rng.random(rows) < 0.2] = 0.0
        k[rng.random(rows) < 0.4] = 0
        p[rng.random(rows) < 0.4] = 1.0
        m[rng.random(rows) < 0.4] = 0.0
    return {"temperature": t, "top_k": k, "top_p": p, "min_p": m, "u": rng.random(rows).astype(np.float32)}


def _tensors(case, seed):
    """The case's inputs as torch tensors on the GPU."""
    gen = _gen(seed)
    if case["op"] == "sample":
        t = {name: torch.from_numpy(a).cuda() for name, a in _settings(case, seed).items()}
        return dict(t, x=_logits(gen, case["rows"], case["n"]))
    heads, kv, hw, ps = (case[key] for key in ("heads", "kv_heads", "width", "page_size"))
    new, lengths = _batch(case)
    per = [-(-n // ps) for n in lengths]
    pages = sum(per) + 3
    order = np.random.default_rng(seed).permutation(pages)
    table = np.zeros((len(new), max(per)), np.int32)  # entries past a sequence's pages are not read
    at = 0
    for s, count in enumerate(per):
        table[s, :count] = order[at:at + count]
        at += count
    dtype, tokens = DTYPES[case["kind"]], sum(new)
    t = {"table": torch.from_numpy(table).cuda(),
         "starts": torch.tensor(np.cumsum([0] + new), dtype=torch.int32).cuda(),
         "lengths": torch.tensor(lengths, dtype=torch.int32).cuda()}
    cache = (pages, kv, ps, hw)
    if case["op"] == "write":
        cos, sin = _rope_tables(max(lengths), hw)
        return dict(t, x=_normal(gen, tokens, heads + 2 * kv, hw), cos=cos, sin=sin,
                    keys=torch.zeros(cache, dtype=dtype, device="cuda"),
                    values=torch.zeros(cache, dtype=dtype, device="cuda"))
    return dict(t, q=_normal(gen, tokens, heads, hw, std=1.5), keys=_normal(gen, *cache).to(dtype),
                values=_normal(gen, *cache).to(dtype))


_device = None


def _dev():
    """The framework's device, and its module (only a tree with the operators has them)."""
    global _device
    if os.path.join(ROOT, "tensomite.cr_amd") not in sys.path:
        sys.path.insert(0, os.path.join(ROOT, "tensomite.cr_amd"))
    import tensomite_hip as th
    if _device is None:
        _device = th.HIPDevice(0)
    return th, _device


def prepare(case, seed):
    t = _tensors(case, seed)
    state = {"case": dict(case), "tensors": t}
    if case["op"] == "sample":
        state["out"] = torch.zeros(case["rows"], dtype=torch.int32, device="cuda")
    else:
        tokens = int(t["starts"][-1])
        shape = (tokens, case["heads"], case["width"])
        state["out"] = torch.zeros(shape, dtype=torch.float32, device="cuda")
        state["new"], state["lengths"] = _batch(case)
    if own:
        th, dev = _dev()
        dev.bind()

        class Borrowed(th.Buffer):
            """A torch tensor's memory as a device buffer: torch keeps owning it."""

            def __init__(self, tensor):
                super().__init__(dev, tensor.data_ptr(), tensor.numel() * tensor.element_size())
                self.tensor = tensor

            def release(self):
                pass

            def __del__(self):
                pass

        b = {name: Borrowed(a) for name, a in t.items()}
        state.update(dev=dev, buffers=b, dst=Borrowed(state["out"]))
        if case["op"] != "sample":
            state["cache"] = dev.paged_cache(case["kind"], t["keys"].shape[0], case["page_size"], case["kv_heads"],
                                             case["width"], keys=b["keys"], values=b["values"])
            state["batch"] = dev.paged_batch(b["table"], t["table"].shape[1], case["sequences"], b["starts"],
                                             b["lengths"], max(state["new"]), max(state["lengths"]))
    torch.cuda.synchronize()
    return state


# ------------------------------------------------------------------- one pass

def run(state):
    case, t = state["case"], state["tensors"]
    op, out = case["op"], state["out"]
    if own:
        dev, b = state["dev"], state["buffers"]
        if op == "sample":
            dev.sample(b["x"], case["rows"], case["n"], b["u"], temperature=b["temperature"], top_k=b["top_k"],
                       top_p=b["top_p"], min_p=b["min_p"], ids=state["dst"])
            return out
        tokens, heads = out.shape[:2]
        if op == "write":
            dev.rope_write_paged(b["x"], (heads + 2 * case["kv_heads"]) * case["width"], tokens, heads, b["cos"],
                                 b["sin"], t["cos"].shape[0], state["cache"], state["batch"], state["dst"])
            return {"q": out, "keys": t["keys"], "values": t["values"]}
        dev.attention_paged(b["q"], tokens, heads, state["cache"], state["batch"], 1.0 / math.sqrt(case["width"]),
                            window=case["window"], sinks=case["sinks"], dst=state["dst"])
        return out
    if op == "sample":
        return _sample(t)
    if op == "write":
        q = _write(case, t, state["new"], state["lengths"])
        return {"q": q, "keys": t["keys"], "values": t["values"]}
    return _attention(case, t, state["new"], state["lengths"], out)


# -------------------------------------------- the plain forms, in elementary torch

def _sample(t):
    x = t["x"].double()
    n = x.shape[1]
    greedy = x.argmax(1)
    sorted_x, order = torch.sort(x, dim=1, descending=True, stable=True)
    temperature = t["temperature"].double()[:, None]
    w = torch.exp((sorted_x - sorted_x[:, :1]) / torch.where(temperature > 0, temperature, 1.0))
    place = torch.arange(n, device=x.device)[None]
    k = t["top_k"][:, None]
    w = torch.where((k <= 0) | (place < k), w, 0.0)
    before = torch.cumsum(w, 1) - w
    p = t["top_p"].double()[:, None]
    w = torch.where((p >= 1.0) | (before < p * w.sum(1, keepdim=True)) | (place == 0), w, 0.0)
    w = torch.where(w >= t["min_p"].double()[:, None], w, 0.0)
    above = torch.cumsum(w, 1) > t["u"].double()[:, None] * w.sum(1, keepdim=True)
    chosen = order.gather(1, above.to(torch.int8).argmax(1, keepdim=True))[:, 0]
    return torch.where(t["temperature"] > 0, chosen, greedy).to(torch.int32)


def _slots(case, t, s, positions):
    """(page, place on it) of sequence s's positions."""
    ps = case["page_size"]
    return t["table"][s][positions // ps].long(), positions % ps


def _write(case, t, new, lengths):
    heads, kv, hw = case["heads"], case["kv_heads"], case["width"]
    x, half = t["x"], hw // 2
    at = torch.cat([torch.arange(n - c, n, device=x.device) for c, n in zip(new, lengths)])
    cos, sin = t["cos"][at][:, None], t["sin"][at][:, None]
    rot = x[:, :heads + kv]
    rot = rot * cos + torch.cat([-rot[..., half:], rot[..., :half]], -1) * sin
    first = 0
    for s, (c, n) in enumerate(zip(new, lengths)):
        page, place = _slots(case, t, s, at[first:first + c])
        t["keys"][page, :, place] = rot[first:first + c, heads:].to(t["keys"].dtype)
        t["values"][page, :, place] = x[first:first + c, heads + kv:].to(t["values"].dtype)
        first += c
    return rot[:, :heads].contiguous()


def _attention(case, t, new, lengths, out):
    heads, kv, hw, window, sinks = (case[key] for key in ("heads", "kv_heads", "width", "window", "sinks"))
    group, q, first = heads // kv, t["q"], 0
    scale = 1.0 / math.sqrt(hw)
    for s, (c, n) in enumerate(zip(new, lengths)):
        low = max(0, n - c - window + 1) if window else 0  # the first position inside any token's window
        at = torch.cat([torch.arange(min(sinks, low), device=q.device), torch.arange(low, n, device=q.device)])
        mine = torch.arange(n - c, n, device=q.device)[:, None]
        seen = at <= mine
        if window:
            seen &= (mine - at < window) | (at < sinks)
        page, place = _slots(case, t, s, at)
        rows = max(1, (1 << 28) // (group * at.numel()))  # query rows at a time: a gigabyte of scores
        for h in range(kv):
            keys, values = t["keys"][page, h, place].float(), t["values"][page, h, place].float()
            for r in range(0, c, rows):
                part = q[first + r:first + min(c, r + rows), h * group:(h + 1) * group]
                scores = part.reshape(-1, hw) @ keys.t().contiguous() * scale
                hide = ~seen[r:r + rows].repeat_interleave(group, 0)
                weights = torch.softmax(scores.masked_fill(hide, -math.inf), -1)
                out[first + r:first + min(c, r + rows), h * group:(h + 1) * group] = \
                    (weights @ values).view(part.shape)
        first += c
    return out


# ---------------------------------------------------------------- what it costs

def _seen(case):
    """Per sequence: (pairs of a new token and a position it sees, positions any of them sees)."""
    window, sinks = case["window"], case["sinks"]
    for c, n in zip(*_batch(case)):
        at = np.arange(n - c, n, dtype=np.int64)
        if not window:
            yield int((at + 1).sum()), n
            continue
        low = np.maximum(0, at - window + 1)
        yield int((at + 1 - low + np.minimum(sinks, low)).sum()), n - int(low[0]) + min(sinks, int(low[0]))


def work(case):
    if case["op"] == "sample":
        size = case["rows"] * case["n"]
        return {"bytes": 4 * size + 24 * case["rows"], "flops": 4 * size}
    heads, kv, hw = case["heads"], case["kv_heads"], case["width"]
    new, lengths = _batch(case)
    tokens, size = sum(new), {"F32": 4, "F16": 2, "BF16": 2}[case["kind"]]
    if case["op"] == "write":
        return {"bytes": tokens * hw * (4 * (heads + 2 * kv) + 4 * heads + 2 * size * kv + 8),
                "flops": 3 * tokens * hw * (heads + kv)}
    seen = list(_seen(case))
    return {"bytes": 8 * tokens * heads * hw + 2 * size * kv * hw * sum(held for _, held in seen),
            "flops": 4 * heads * hw * sum(pairs for pairs, _ in seen)}


# ------------------------------------------------------- the definitions in 64 bits

def _exact_token(x, t, k, p, m, u):
    """One row on the host: candidates in falling order (the lower index first), cut by top-k, top-p and min-p."""
    if not t > 0.0:
        return int(np.argmax(x))
    order = np.lexsort((np.arange(x.size), -x))
    if 0 < k < x.size:
        order = order[:k]
    w = np.exp((x[order] - x[order[0]]) / np.float64(t))
    if p < 1.0:
        order = order[:max(1, int(np.searchsorted(np.cumsum(w), np.float64(p) * w.sum())) + 1)]
        w = w[:order.size]
    w = w[w >= np.float64(m)]
    return int(order[min(int(np.searchsorted(np.cumsum(w), np.float64(u) * w.sum(), side="right")), w.size - 1)])


def _exact_attention(case, t):
    heads, kv, hw, ps = (case[key] for key in ("heads", "kv_heads", "width", "page_size"))
    window, sinks, group = case["window"], case["sinks"], heads // kv
    outs, first = [], 0
    for s, (c, n) in enumerate(zip(*_batch(case))):
        out = torch.empty(c, heads, hw, dtype=torch.float64, device="cuda")
        pages = t["table"][s, :-(-n // ps)].long()
        rows = max(1, (1 << 27) // n)
        for h in range(heads):
            keys = t["keys"][pages, h // group].reshape(-1, hw)[:n].double()
            values = t["values"][pages, h // group].reshape(-1, hw)[:n].double()
            for r in range(0, c, rows):
                end = min(c, r + rows)
                score = (t["q"][first + r:first + end, h].double() @ keys.T.contiguous()) / math.sqrt(hw)
                mine = torch.arange(n - c + r, n - c + end, device="cuda")[:, None]
                at = torch.arange(n, device="cuda")[None]
                hidden = at > mine
                if window:
                    hidden = hidden | ((at <= mine - window) & (at >= sinks))
                score[hidden] = -math.inf
                e = torch.exp(score - score.amax(1, keepdim=True))
                out[r:end, h] = (e @ values) / e.sum(1, keepdim=True)
        outs.append(out)
        first += c
    return torch.cat(outs)


def _exact_write(case, t):
    heads, kv, ps = case["heads"], case["kv_heads"], case["page_size"]
    x = t["x"].double()
    left, right = x[..., :case["width"] // 2], x[..., case["width"] // 2:]
    keys, values = t["keys"].double(), t["values"].double()
    q, first = torch.empty_like(x[:, :heads]), 0
    for s, (c, n) in enumerate(zip(*_batch(case))):
        rows = slice(first, first + c)
        cos, sin = t["cos"][n - c:n].double()[:, None], t["sin"][n - c:n].double()[:, None]
        turned = x[rows] * cos + torch.cat([-right[rows], left[rows]], -1) * sin
        q[rows] = turned[:, :heads]
        at = torch.arange(n - c, n, device="cuda")
        page = t["table"][s, at // ps].long()
        keys[page, :, at % ps] = turned[:, heads:heads + kv]
        values[page, :, at % ps] = x[rows, heads + kv:]
        first += c
    return {"q": q, "keys": keys, "values": values}


def exact(case, seed):
    t = _tensors(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, t)
    if case["op"] == "write":
        return _exact_write(case, t)
    x = t["x"].double().cpu().numpy()
    s = _settings(case, seed)
    return torch.tensor([_exact_token(x[r], s["temperature"][r], s["top_k"][r], s["top_p"][r], s["min_p"][r],
                                      s["u"][r]) for r in range(case["rows"])], dtype=torch.int32)
