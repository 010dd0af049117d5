"""Cases that time the serving operators: attention for rows that share a long prefix, attention with a sliding window
and sinks (single tokens and a prompt's chunk), beam search's selection, and the reordering of its sequences' caches.

Each case is a dict of plain values. `prepare` makes what a program holds before the call, `run` makes one call: with
`own` the framework's operator on device addresses, otherwise the same in elementary torch operations. `exact` computes
it in 64 bits and `work` says what the call cannot do without.

The kinds of call:
  rows     one token of each of n sequences against its cache (va.attention_rows). Groups of `group` sequences share
           their first `shared` positions, which lie in one of them; each has up to `longest` positions of its own
           behind those. `window` > 0: a row sees its last `window` positions and the first `sinks`
  run      n consecutive tokens of one sequence from position `at`, a prompt's chunk (va.attention_run)
  select   the `keep` best of each group's `width` beams x `vocab` continuations (va.beam_select)
  reorder  the caches of each group's beams after a selection, in every layer (va.kv_reorder): a beam that continues
           stays where it is, one that ended takes over the positions since the prompt of one that continues twice

Caches are [sequence][layer][position][key-value head x dimension], as the engine's are.
"""
import math
import os
import sys

import torch

DEV = "cuda" if torch.cuda.is_available() else "cpu"
own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _rows(n, heads, kv_heads, dim, dtype, longest, shared=0, group=1, window=0, sinks=0):
    return dict(kind="rows", n=n, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, longest=longest, shared=shared, group=group,
                window=window, sinks=sinks)


def _run(n, at, heads, kv_heads, dim, dtype, window, sinks):
    return dict(kind="run", n=n, at=at, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, window=window, sinks=sinks)


def _select(groups, width, vocab, keep):
    return dict(kind="select", groups=groups, width=width, vocab=vocab, keep=keep)


def _reorder(groups, width, layers, kv_heads, dim, dtype, prompt, longest):
    return dict(kind="reorder", groups=groups, width=width, layers=layers, kv_heads=kv_heads, dim=dim, dtype=dtype, prompt=prompt,
                longest=longest)


def listed():
    return [
        # four beams of a chat's short prompt: launches and latency
        dict(_rows(4, 32, 4, 128, "f32", 40, shared=777, group=4), name="shared_4_of_777"),
        # the benchmark's batch of 32 sequences, all behind one long system prompt
        dict(_rows(32, 32, 4, 128, "f32", 256, shared=8192, group=32), name="shared_32_of_8k"),
        # five prompts with eight answers each, a key-value head for every head, a bfloat16 cache
        dict(_rows(40, 16, 16, 128, "bf16", 333, shared=2048, group=8), name="shared_5x8_bf16"),
        # a chat's token far into its context: the last 1024 positions and four sinks
        dict(_rows(1, 32, 4, 128, "f32", 8100, window=1024, sinks=4), name="window_token"),
        # a batch of ragged sequences with a wide window, a half-precision cache
        dict(_rows(32, 32, 4, 128, "f16", 8192, window=4096, sinks=4), name="window_batch_f16"),
        # a short chunk of a prompt on small heads, an odd number of rows, a narrow window
        dict(_run(333, 1500, 8, 2, 64, "bf16", 500, 5), name="window_prompt_333"),
        # a full chunk of a long prompt
        dict(_run(1024, 7168, 32, 4, 128, "f32", 4096, 4), name="window_prompt_1024"),
        # one prompt's four beams over the benchmark's vocabulary
        dict(_select(1, 4, 151936, 8), name="select_4"),
        # a server's eight prompts with eight beams each
        dict(_select(8, 8, 151936, 16), name="select_8x8"),
        # wide beams over a small odd vocabulary
        dict(_select(3, 32, 40001, 64), name="select_3x32_wide"),
        # four beams a few hundred tokens behind their prompt, a small model's layers
        dict(_reorder(1, 4, 4, 4, 128, "f32", 777, 300), name="reorder_4"),
        # eight prompts' eight beams each, half the benchmark model's layers
        dict(_reorder(8, 8, 24, 4, 128, "f32", 64, 256), name="reorder_8x8"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["shared", "shared", "window", "window", "run", "run", "select", "select", "reorder"])
    heads, kv_heads, dim = rng.choice([(32, 4, 128), (32, 4, 128), (16, 16, 128), (16, 4, 128), (8, 2, 64), (6, 2, 128), (12, 4, 64)])
    dtype = rng.choice(["f32", "f32", "f16", "bf16"])
    if kind == "shared":
        group = _log(rng, 1, 32)
        n = group * rng.randint(1, max(1, 40 // group))
        return _rows(n, heads, kv_heads, dim, dtype, _log(rng, 1, 400), shared=_log(rng, 16, 8192 * 4 // max(4, n // group)), group=group,
                     window=rng.choice([0, 0, 0, _log(rng, 64, 2000)]), sinks=rng.randint(0, 8))
    if kind == "window":
        return _rows(_log(rng, 1, 32), heads, kv_heads, dim, dtype, _log(rng, 64, 8192 if kv_heads < 16 else 3000),
                     window=_log(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 4, 16, 100]))
    if kind == "run":
        return _run(_log(rng, 2, 1024), rng.choice([0, rng.randint(1, 7000)]), heads, kv_heads, dim, dtype, _log(rng, 1, 4096),
                    rng.choice([0, 1, 4, 4, 16, 100]))
    if kind == "select":
        width = _log(rng, 1, 32)
        return _select(rng.randint(1, max(1, 64 // width)), width, rng.choice([1000, 40000, 151936, _log(rng, 100, 150000)]),
                       min(64, rng.choice([width, 2 * width, 1, _log(rng, 1, 64)])))
    width = _log(rng, 2, 32)
    return _reorder(rng.randint(1, max(1, 64 // width)), width, _log(rng, 1, 24 if kv_heads <= 4 else 6), kv_heads, dim, dtype, rng.randint(0, 100), _log(rng, 1, 200))


# --- inputs -----------------------------------------------------------------------------------------------------------

class State:
    pass


def _generator(seed, what):
    g = torch.Generator(device=DEV)
    g.manual_seed((seed * 1000003 + what) % (1 << 62))
    return g


def _randn(shape, seed, what, dtype=torch.float32):
    return torch.randn(shape, generator=_generator(seed, what), device=DEV, dtype=torch.float32).to(dtype)


def _uniform(low, high, shape, seed, what):
    """Whole numbers low .. high."""
    return torch.randint(low, high + 1, shape, generator=_generator(seed, what), device=DEV, dtype=torch.int32)


def _survivors(groups, width, seed):
    """Each beam's parent in its group: a beam that some continuation came from is its own, the others take one of those."""
    chosen = _uniform(0, width - 1, (groups, width), seed, 7).long()
    lives = torch.zeros((groups, width), dtype=torch.bool, device=DEV)
    lives.scatter_(1, chosen, True)
    itself = torch.arange(width, device=DEV).expand(groups, width)
    return torch.where(lives, itself, chosen).int().contiguous()


def prepare(case, seed):
    s = State()
    s.case, kind = case, case["kind"]
    if kind in ("rows", "run"):
        n, heads, kv_heads, dim, dtype = case["n"], case["heads"], case["kv_heads"], case["dim"], TYPES[case["dtype"]]
        s.scale = 1.0 / math.sqrt(dim)
        # queries and keys are normalized by head, so their scores are a few units wide
        s.q = _randn((n, heads, dim), seed, 1) * 1.5
        if kind == "rows":
            s.seqs, s.ctx = n, case["shared"] + case["longest"]
            mine = torch.arange(n, device=DEV, dtype=torch.int32)
            ahead = _uniform(min(case["longest"], 1 if case["shared"] else max(1, case["longest"] // 8)), case["longest"], (n,), seed, 2)
            s.rows = torch.stack([mine, case["shared"] + ahead - 1, mine // case["group"] * case["group"],
                                  torch.full_like(mine, case["shared"])], 1).contiguous()
        else:
            s.seqs, s.ctx = 2, case["at"] + n
        s.k = _randn((s.seqs, 1, s.ctx, kv_heads, dim), seed, 3, dtype)
        s.v = _randn((s.seqs, 1, s.ctx, kv_heads, dim), seed, 4, dtype)
        s.out = torch.empty((n, heads, dim), device=DEV)
    elif kind == "select":
        rows = case["groups"] * case["width"]
        # a model's logits: a broad bulk, and a few tokens well above it
        s.logits = _randn((rows, case["vocab"]), seed, 1) * 2.0
        at = torch.randint(0, case["vocab"], (rows, 40), generator=_generator(seed, 2), device=DEV)
        s.logits.scatter_add_(1, at, 6.0 + 3.0 * _randn((rows, 40), seed, 3))
        s.scores = -20.0 + 1.5 * _randn((rows,), seed, 4)
        s.ended = (_uniform(0, 15, (rows,), seed, 5) == 0).to(torch.uint8)
        s.end = case["vocab"] - 1
        s.best = torch.empty((case["groups"], case["keep"]), device=DEV)
        s.parents = torch.empty((case["groups"], case["keep"]), dtype=torch.int32, device=DEV)
        s.tokens = torch.empty((case["groups"], case["keep"]), dtype=torch.int32, device=DEV)
    else:
        groups, width = case["groups"], case["width"]
        s.seqs, s.ctx = groups * width, case["prompt"] + case["longest"]
        shape = (s.seqs, case["layers"], s.ctx, case["kv_heads"], case["dim"])
        s.k = _randn(shape, seed, 1, TYPES[case["dtype"]])
        s.v = _randn(shape, seed, 2, TYPES[case["dtype"]])
        s.order = torch.arange(s.seqs, device=DEV, dtype=torch.int32)
        s.parents = _survivors(groups, width, seed)
        ahead = _uniform((case["longest"] + 1) // 2, case["longest"], (groups,), seed, 8)
        s.spans = torch.stack([torch.full_like(ahead, case["prompt"]), case["prompt"] + ahead], 1).contiguous()
    s.work = torch.empty(256 << 20, dtype=torch.uint8, device=DEV)  # a program's workspace for all of them
    s.view = None
    return s


# --- calls ------------------------------------------------------------------------------------------------------------

def run(s):
    if own:
        return _own(s)
    kind = s.case["kind"]
    if kind == "rows":
        return _plain_rows(s)
    if kind == "run":
        return _plain_run(s)
    if kind == "select":
        return _plain_select(s)
    return _plain_reorder(s)


def _own(s):
    path = os.path.join(os.getcwd(), "vitna-anchor_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import vitna_amd as va
    case, stream = s.case, torch.cuda.current_stream().cuda_stream if DEV == "cuda" else 0
    if case["kind"] != "select":
        layers, width = case.get("layers", 1), case["kv_heads"] * case["dim"]
        if s.view is None:  # a program describes its cache once
            dtype = {"f32": va.F32, "f16": va.F16, "bf16": va.BF16}[case["dtype"]]
            s.view = va.kv_view(s.k.data_ptr(), s.v.data_ptr(), dtype, case.get("heads", case["kv_heads"]), case["kv_heads"], case["dim"],
                                s.ctx, s.seqs, seq_stride=layers * s.ctx * width, window=case.get("window", 0), sinks=case.get("sinks", 0))
    if case["kind"] == "rows":
        va.attention_rows(s.view, s.q.data_ptr(), s.rows.data_ptr(), case["n"], s.out.data_ptr(), s.work.data_ptr(), s.work.numel(),
                          own_max=case["longest"], shared_max=case["shared"], stream=stream)
        return s.out
    if case["kind"] == "run":
        va.attention_run(s.view, 1, case["at"], s.q.data_ptr(), case["n"], s.out.data_ptr(), s.work.data_ptr(), s.work.numel(), stream=stream)
        return s.out
    if case["kind"] == "select":
        va.beam_select(s.logits.data_ptr(), case["vocab"], case["groups"], case["width"], case["keep"], s.scores.data_ptr(),
                       s.best.data_ptr(), s.parents.data_ptr(), s.tokens.data_ptr(), s.work.data_ptr(), s.work.numel(),
                       ended=s.ended.data_ptr(), end_token=s.end, stream=stream)
        return s.best, s.parents, s.tokens
    va.kv_reorder(s.view, layers, s.ctx * width, s.order.data_ptr(), s.parents.data_ptr(), s.spans.data_ptr(), case["groups"], case["width"],
                  longest=case["longest"], stream=stream)
    return s.k, s.v


def _attend(q, k, v, visible, scale):
    """softmax(q k) v over the visible positions: q [..., queries, dim], k and v [..., positions, dim]. Zeros where none is."""
    score = (torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale).masked_fill(~visible, -math.inf)
    most = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(most == -math.inf, torch.zeros_like(most), most))
    total = weight.sum(-1, keepdim=True)
    return torch.matmul(weight / torch.where(total == 0, torch.ones_like(total), total), v)


def _seen(pos, t, window, sinks):
    before = t <= pos
    return before & ((t > pos - window) | (t < sinks)) if window else before


def _plain_rows(s):
    case = s.case
    n, heads, kv_heads, dim = case["n"], case["heads"], case["kv_heads"], case["dim"]
    t = torch.arange(s.ctx, device=DEV)
    rows = s.rows.long()
    seq, pos, base, shared = rows[:, 0:1], rows[:, 1:2], rows[:, 2:3], rows[:, 3:4]
    source = torch.where(t < shared, base, seq)
    k = s.k[source, 0, t].float().transpose(1, 2).contiguous()  # [n, kv head, position, dim]
    v = s.v[source, 0, t].float().transpose(1, 2).contiguous()
    visible = _seen(pos, t, case["window"], case["sinks"])[:, None, None, :]
    out = _attend(s.q.view(n, kv_heads, heads // kv_heads, dim), k, v, visible, s.scale)
    return out.reshape(n, heads, dim)


def _plain_run(s):
    case = s.case
    n, heads, kv_heads, dim = case["n"], case["heads"], case["kv_heads"], case["dim"]
    group = heads // kv_heads
    t = torch.arange(case["at"] + n, device=DEV)
    pos = case["at"] + torch.arange(n, device=DEV)
    k = s.k[1, 0, :case["at"] + n].float().transpose(0, 1).contiguous()  # [kv head, position, dim]
    v = s.v[1, 0, :case["at"] + n].float().transpose(0, 1).contiguous()
    q = s.q.view(n, kv_heads, group, dim).permute(1, 2, 0, 3).reshape(kv_heads, group * n, dim)
    visible = _seen(pos[:, None], t, case["window"], case["sinks"]).repeat(group, 1)
    out = _attend(q, k, v, visible, s.scale)
    return out.view(kv_heads, group, n, dim).permute(2, 0, 1, 3).reshape(n, heads, dim)


def _plain_select(s):
    groups, width, vocab, keep = s.case["groups"], s.case["width"], s.case["vocab"], s.case["keep"]
    # in 64 bits: two beams' sums lie near each other, and which is larger decides
    x = s.logits.double()
    most = x.amax(1, keepdim=True)
    value = s.scores.double()[:, None] + ((x - most) - torch.log(torch.exp(x - most).sum(1, keepdim=True)))
    ended = (s.ended != 0)[:, None]
    at_end = torch.arange(vocab, device=DEV)[None, :] == s.end
    value = torch.where(ended, torch.where(at_end, s.scores.double()[:, None], -math.inf), value)
    best, index = torch.sort(value.view(groups, width * vocab), dim=1, descending=True, stable=True)
    best, index = best[:, :keep], index[:, :keep]
    none = best == -math.inf
    parents = torch.where(none, -1, index // vocab).int()
    tokens = torch.where(none, -1, index % vocab).int()
    return best.float(), parents, tokens


def _plain_reorder(s):
    case = s.case
    width, first = case["width"], case["prompt"]
    beams = torch.arange(s.seqs, device=DEV)
    source = s.order.long()[beams // width * width + s.parents.view(-1).long()]
    t = torch.arange(first, s.ctx, device=DEV)
    spans = s.spans.long()[beams // width]
    inside = ((t >= spans[:, 0:1]) & (t < spans[:, 1:2]))[:, None, :, None, None]
    s.k[:, :, first:] = torch.where(inside, s.k[source][:, :, first:], s.k[:, :, first:])
    s.v[:, :, first:] = torch.where(inside, s.v[source][:, :, first:], s.v[:, :, first:])
    return s.k, s.v


# --- what a call needs ------------------------------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "select":
        rows = case["groups"] * case["width"]
        return {"bytes": 4.0 * rows * case["vocab"] + 5.0 * rows + 12.0 * case["groups"] * case["keep"], "flops": 3.0 * rows * case["vocab"]}
    size = 4.0 if case["dtype"] == "f32" else 2.0
    position = 2.0 * size * case["kv_heads"] * case["dim"]  # a position's keys and values
    if kind == "reorder":
        # of `width` beams with a random parent each, (1 - 1 / width) ^ width end; each that ends is written, and the
        # beams that they take over from are read
        ends = case["width"] * (1.0 - 1.0 / case["width"]) ** case["width"]
        read = min(ends, case["width"] - ends)
        return {"bytes": case["groups"] * (ends + read) * case["layers"] * 0.75 * case["longest"] * position, "flops": 0.0}
    n, heads, dim = case["n"], case["heads"], case["dim"]
    ends = 2.0 * 4.0 * n * heads * dim  # queries and outputs
    if kind == "run":
        at = case["at"]
        first = max(0, at - case["window"] + 1)
        read = at + n - first + min(case["sinks"], first)
        seen = sum(min(p + 1, case["window"] + min(case["sinks"], max(0, p + 1 - case["window"]))) for p in range(at, at + n))
        return {"bytes": read * position + ends, "flops": 4.0 * seen * heads * dim}
    longest, shared, window, sinks = case["longest"], case["shared"], case["window"], case["sinks"]
    mine = (min(longest, 1 if shared else max(1, longest // 8)) + longest) / 2.0
    if window:
        before = max(0.0, min(float(shared), window - mine)) + min(sinks, shared)  # of the prefix
        mine = min(mine, window + (0 if shared else sinks))
    else:
        before = float(shared)
    return {"bytes": (n / case["group"] * before + n * mine) * position + ends, "flops": 4.0 * n * (before + mine) * heads * dim}


# --- the same in 64 bits ----------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "reorder":
        return None  # values moved, none computed
    if kind == "select":
        best = []
        for g in range(case["groups"]):
            values = []
            for b in range(g * case["width"], (g + 1) * case["width"]):
                if s.ended[b]:
                    values.append(s.scores[b:b + 1].double())
                else:
                    values.append(s.scores[b].double() + torch.log_softmax(s.logits[b].double(), 0))
            values = torch.cat(values)
            top = torch.topk(values, min(case["keep"], values.numel())).values
            best.append(torch.cat([top, torch.full((case["keep"] - top.numel(),), -math.inf, dtype=torch.float64, device=DEV)]))
        return torch.stack(best), None, None
    n, heads, kv_heads = case["n"], case["heads"], case["kv_heads"]
    out = torch.zeros((n, heads, case["dim"]), dtype=torch.float64, device=DEV)
    window = case["window"] or 1 << 30

    def head(q, k, v, pos, first):
        """One head: q [queries, dim] at positions pos against positions first .. of k and v."""
        t = torch.arange(first, first + k.shape[0], device=DEV)[None, :]
        hidden = (t > pos[:, None]) | ((t <= pos[:, None] - window) & (t >= case["sinks"]))
        score = (q.double() @ k.double().t()) / math.sqrt(case["dim"])
        return torch.softmax(score.masked_fill(hidden, -math.inf), -1) @ v.double()

    if kind == "run":
        pos = torch.arange(case["at"], case["at"] + n, device=DEV)
        for h in range(heads):
            kv = h * kv_heads // heads
            out[:, h] = head(s.q[:, h], s.k[1, 0, :, kv], s.v[1, 0, :, kv], pos, 0)
        return out
    for i, (seq, pos, base, shared) in enumerate(s.rows.tolist()):
        k = torch.cat([s.k[base, 0, :shared], s.k[seq, 0, shared:pos + 1]])
        v = torch.cat([s.v[base, 0, :shared], s.v[seq, 0, shared:pos + 1]])
        at = torch.full((heads // kv_heads,), pos, device=DEV)
        for kv in range(kv_heads):
            mine = slice(kv * heads // kv_heads, (kv + 1) * heads // kv_heads)
            out[i, mine] = head(s.q[i, mine], k[:, kv], v[:, kv], at, 0)
    return out
