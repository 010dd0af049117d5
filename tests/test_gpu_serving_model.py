"""A model's serving calls (include/vitna_serve.h): a sliding window on every path, sequences that share a prefix, and beam
search.

The attention of a row is checked at the last layer against 64-bit numpy on the device's own queries and cache: its
scores carry float32's roundings of the query's norm and rotation (some 2^-22 of a score) beside the kernels' own
(2^-20 of a product at most), which leaves 1e-6 of the outputs' 2-norm at random; 2e-5 is asked for.
Logits of two passes that differ in such roundings go apart in what follows: the multi-row projections take activations
in two bfloat16 parts, and inputs that differ in their last bit are cut differently. A product so cut is 4.2e-6 off at
random (0.4 2^-8 a part, squared, three such terms); a layer has five in a row (q/k/v, o, router's input and gate/up,
down, and the residual's norm before them) and the head one, so two layers leave sqrt(11) 4.2e-6 = 1.4e-5 of the logits in
each pass and sqrt(2) times that, 2e-5, between two; twice that is asked for. (1e-5, which stood here first, forgot the
second pass and the chain: 1.05e-5 was seen.)
"""
import numpy as np
import pytest

import vitna_amd as va
from test_gpu_serving import select_want, visible

pytestmark = pytest.mark.gpu

SPECS = {
    "g4": dict(n_layers=2, hidden=512, intermediate=256, n_heads=8, n_kv_heads=2, head_dim=128, vocab=1000, n_experts=32, n_experts_used=8,
               renormalize=1, norm_std=0.1, ctx=700, seqs=12, kv_host=0),
    "g8": dict(n_layers=2, hidden=512, intermediate=256, n_heads=16, n_kv_heads=2, head_dim=128, vocab=1000, n_experts=16, n_experts_used=4,
               renormalize=1, norm_std=0.1, ctx=700, seqs=12, kv_host=0),
    "hd64": dict(n_layers=1, hidden=512, intermediate=256, n_heads=8, n_kv_heads=8, head_dim=64, vocab=1000, n_experts=16, n_experts_used=4,
                 renormalize=1, norm_std=0.1, ctx=700, seqs=12, kv_host=0),
}


class Pair:
    """A model on the device (or twice), its caches filled alike."""

    def __init__(self, name, many=1, **kw):
        self.model = va.Model(va.shape(**dict(SPECS[name], **kw)), 31)
        self.devs = [va.Device(self.model) for _ in range(many)]
        for d in self.devs:
            d.kv_fill(5, [self.model.m.ctx] * self.model.m.seqs)
        self.tabs = [t.astype(np.float64) for t in self.model.rope_tables()]

    def __enter__(self):
        return (self, *self.devs)

    def __exit__(self, *_):
        for d in self.devs:
            d.close()
        self.model.free()

    def attention(self, dev, q, row, window, sinks):
        """The attention of a row (token, pos, seq) at the last layer, from its raw query, in 64 bits."""
        cfg = self.model.cfg
        hd, G, layer = cfg.head_dim, cfg.n_heads // cfg.n_kv_heads, cfg.n_layers - 1
        w = np.ctypeslib.as_array(self.model.m.layers[layer].q_norm, shape=(hd,)).astype(np.float64)
        x = q.astype(np.float64).reshape(cfg.n_heads, hd)
        x = x / np.sqrt((x * x).mean(1, keepdims=True) + cfg.rms_eps) * w
        c, s = self.tabs[0][row[1]], self.tabs[1][row[1]]
        a, b = x[:, :hd // 2], x[:, hd // 2:]
        x = np.concatenate([a * c - b * s, b * c + a * s], 1)
        k, v = dev.kv(row[2], layer, 0, row[1] + 1)
        t = visible(row[1], window, sinks)
        k = k.reshape(-1, cfg.n_kv_heads, hd)[t].astype(np.float64)
        v = v.reshape(-1, cfg.n_kv_heads, hd)[t].astype(np.float64)
        out = np.empty((cfg.n_heads, hd))
        for h in range(cfg.n_heads):
            sc = k[:, h // G] @ x[h] / np.sqrt(hd)
            p = np.exp(sc - sc.max())
            out[h] = p / p.sum() @ v[:, h // G]
        return out.ravel()

    def check(self, dev, rows, window, sinks, some=None):
        for i in range(len(rows)) if some is None else some:
            q, att = dev.attention_io(i)
            want = self.attention(dev, q, rows[i], window, sinks)
            rel = np.linalg.norm(att - want) / np.linalg.norm(want)
            assert rel <= 2e-5, (i, rows[i], rel)


def near(a, b):
    assert np.max(np.abs(a.astype(np.float64) - b)) <= 4e-5 * np.max(np.abs(b))


@pytest.mark.parametrize("name", list(SPECS))
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 4), (150, 70), (699, 0)])
def test_window_on_every_path(name, window, sinks):
    with Pair(name) as (pair, dev):
        dev.set_window(window, sinks)
        for pos in (0, 1, 63, 64, 300, 699):
            row = (7 + pos, pos, 3)
            dev.step(row[2], row[0], row[1])
            pair.check(dev, [row], window, sinks)
        rows = [(11 * i, (97 * i + 5) % 700, i) for i in range(12)]
        dev.rows_step(rows)
        pair.check(dev, rows, window, sinks)
        rows = [(i, 200 + i, 5) for i in range(90)]  # a prompt's chunk
        dev.rows_step(rows)
        pair.check(dev, rows, window, sinks, [0, 1, 31, 32, 63, 64, 89])
        rows = [(i, 3 + i, 6) for i in range(7)] + [(9, 640, 2)]  # drafts of one sequence and another's token
        for rows in (rows, rows[:7], rows[7:]):
            for layer in range(pair.model.cfg.n_layers):
                lg = dev.rows_route(rows, layer)
                if layer + 1 < pair.model.cfg.n_layers:
                    r = [va.host_route(x, pair.model.cfg.n_experts_used, True) for x in lg]
                    dev.rows_experts(layer, np.stack([x[1] for x in r]), np.stack([x[2] for x in r]))
            pair.check(dev, rows, window, sinks)


def test_a_window_over_a_long_cache():
    """A chunk in a cache so long that images of all of it are more than the call takes, at a position where they are not."""
    with Pair("g4", n_layers=1, n_heads=32, n_kv_heads=16, ctx=20000, seqs=1) as (pair, dev):
        dev.set_window(4096, 4)
        rows = [(i % 1000, 7168 + i, 0) for i in range(1024)]
        dev.rows_step(rows)
        pair.check(dev, rows, 4096, 4, [0, 700, 1023])


def test_a_prefix_near_the_caches_end():
    """Rows behind a prefix whose power of two lies past the cache."""
    with Pair("g4") as (pair, dev):
        dev.kv_fork(2, 650, [5, 0, 7])
        rows = [(3 + i, 690 + i, s) for i, s in enumerate((2, 5, 0, 7))]
        dev.rows_step(rows)
        dev.set_exact_rows(0)
        dev.rows_step(rows)
        pair.check(dev, rows, 0, 0)


def test_window_taken_away():
    """window 0, or as long as the cache, is the model as it was, bit for bit; a changed window is honoured by graphs made
    before; the persistent step is not taken with one."""
    with Pair("g4") as (pair, dev):
        rows = [(11 * i, (97 * i + 5) % 700, i) for i in range(12)]
        before = dev.step(3, 9, 400), dev.rows_step(rows)
        for window, sinks in ((100, 4), (100, 5), (30, 0)):
            dev.set_window(window, sinks)
            taken = dev.set_step_kernel(True)
            assert not taken
            dev.step(3, 9, 400)
            pair.check(dev, [(9, 400, 3)], window, sinks)
            for shift in (0, 1, 2):  # replays
                dev.rows_step([(t, (p + shift) % 700, s) for t, p, s in rows])
                pair.check(dev, [(t, (p + shift) % 700, s) for t, p, s in rows], window, sinks)
        dev.set_step_kernel(False)
        for window in (0, 700, 10 ** 9):
            dev.set_window(64, 4)
            dev.set_window(window, 4)
            dev.kv_fill(5, [700] * 12)
            after = dev.step(3, 9, 400), dev.rows_step(rows)
            assert all(np.array_equal(x.view(np.uint32), y.view(np.uint32)) for x, y in zip(before, after))


@pytest.mark.parametrize("name", list(SPECS))
def test_window_passes_keep_a_steps_bits(name):
    """A pass of few rows gives each row the logits bits of its own step, with a window too."""
    rows = [(5 + i, 100 + i, 4) for i in range(6)] + [(60, 699, 1), (61, 0, 2), (62, 350, 3)]
    with Pair(name, 2) as (pair, a, b):
        cfg = pair.model.cfg
        for d in (a, b):
            d.set_window(77, 4)
        for layer in range(cfg.n_layers):
            lg = a.rows_route(rows, layer)
            r = [va.host_route(x, cfg.n_experts_used, True) for x in lg]
            a.rows_experts(layer, np.stack([x[1] for x in r]), np.stack([x[2] for x in r]))
        got = a.rows_head(len(rows))
        for i, (token, pos, seq) in enumerate(rows):
            for layer in range(cfg.n_layers):
                _, order, weights = va.host_route(b.moe_route(seq, token, pos, layer), cfg.n_experts_used, True)
                b.moe_experts(layer, order, weights)
            assert np.array_equal(got[i].view(np.uint32), b.moe_head().view(np.uint32)), i


@pytest.mark.parametrize("name", list(SPECS))
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 4)])
def test_forked_sequences(name, window, sinks):
    """Rows of sequences that share a prefix: the logits of sequences that hold copies of it; the prefix's caches in every
    layer; several groups, rows without one, and replays as the sequences grow."""
    with Pair(name, 2) as (pair, a, b):
        L = pair.model.cfg.n_layers
        for d in (a, b):
            d.set_window(window, sinks)
        a.kv_fork(0, 333, [3, 1, 2])
        a.kv_fork(4, 64, [5])
        a.kv_fork(3, 200, [6])  # of a sequence that shares already: the same base, a shorter prefix
        for dst, src, n in ((3, 0, 333), (1, 0, 333), (2, 0, 333), (5, 4, 64), (6, 0, 200)):
            for layer in range(L):
                b.kv(dst, layer, 0, n, *b.kv(src, layer, 0, n))
                got, want = a.kv(dst, layer, 0, 700), b.kv(dst, layer, 0, 700)
                assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
        for turn in range(4):
            rows = [(turn + 3 * s, 333 + turn + 5 * i, s) for i, s in enumerate((0, 1, 2, 3))] + [(9, 64 + turn, 4), (10, 70 + turn, 5), (11, 200 + turn, 6), (12, 600, 7)]
            near(a.rows_step(rows), b.rows_step(rows))
            pair.check(a, rows, window, sinks)


def test_forked_sequences_that_change():
    """A prefix is shared up to where one of its sequences has changed it, whichever; other paths see the copies."""
    with Pair("g4") as (pair, dev):
        seqs = [0, 1, 2, 3]

        def look(*at):
            rows = [(5 + s, 400 + s, s) for s in seqs]
            dev.rows_step(rows)
            pair.check(dev, rows, 0, 0)

        dev.kv_fork(0, 300, [1, 2, 3])
        look()
        dev.rows_step([(7, 250, 2), (8, 500, 1)])  # a row inside the prefix of one
        look()
        k, v = dev.kv(0, 1, 100, 4)
        dev.kv(0, 1, 100, 4, k + 1, v - 1)  # the base's own
        look()
        dev.step(0, 3, 50)
        look()
        dev.kv_fork(3, 350, [0, 1, 2])  # another base
        look()
        dev.kv_fork(2, 20, [3])
        look()
        dev.kv_fill(6, [700] * 12)
        look()
        dev.kv_fork(5, 700, [6])
        rows = [(1, 699, 5), (2, 699, 6)]
        dev.rows_step(rows)
        pair.check(dev, rows, 0, 0)
        rows = [(i, 320 + i, 6) for i in range(80)]  # a chunk of a sequence that shares
        dev.rows_step(rows)
        pair.check(dev, rows, 0, 0, [0, 33, 79])


def host_beams(dev, layers, prompt_rows, groups, width, steps, end, seqs):
    """Beam search with every beam's whole cache moved by the host after each step; with the scores, how far another pass
    may leave them: a step's logits lie within 4e-5 of the largest, a score adds one and the log of their sum, and takes over
    its parent's."""
    rows, scores, ended = list(prompt_rows), np.full(groups * width, -np.inf, np.float32), np.zeros(groups * width, np.uint8)
    scores[::width] = 0.0
    log, off = [], 0.0
    for _ in range(steps):
        logits = dev.rows_step(rows)
        off += 2 * 4e-5 * float(np.max(np.abs(logits)))
        best, par, tok = select_want(logits, scores, ended if end >= 0 else None, max(end, 0), groups, width, width)
        top = max(r[1] for r in rows) + 1
        old = {r[2]: [dev.kv(r[2], layer, 0, top) for layer in range(layers)] for r in rows}
        nxt, nsc, nen, npar = [], [], [], []
        for g in range(groups):
            for j in range(width):
                p = par[g, j]
                src = rows[g * width + p]
                here = seqs[g * width + j]
                for layer in range(layers):
                    dev.kv(here, layer, 0, top, *old[src[2]][layer])
                over = bool(ended[g * width + p])
                nxt.append((int(tok[g, j]), src[1] + (0 if over else 1), here))
                nen.append(over or tok[g, j] == end)
                nsc.append(best[g, j])
                npar.append(p)
        rows, scores, ended = nxt, np.array(nsc, np.float32), np.array(nen, np.uint8)
        log.append((list(npar), [r[0] for r in rows], scores.copy(), off))
    return log


@pytest.mark.parametrize("name,groups,width,end", [("g4", 1, 4, -1), ("g4", 2, 3, -1), ("g8", 2, 5, 17), ("hd64", 1, 12, -1), ("g4", 3, 1, -1)])
def test_beam_steps(name, groups, width, end):
    """Parents, tokens and scores of every step, as a search whose caches the host moves whole."""
    n, steps, before = groups * width, 8, 130
    with Pair(name, 2) as (pair, a, b):
        L = pair.model.cfg.n_layers
        prompts = [11 * g for g in range(groups)]
        seqs = [(5 * i + 2) % 12 for i in range(n)]
        for g in range(groups):
            mine = seqs[g * width:(g + 1) * width]
            a.kv_fork(mine[0], before, mine[1:])
            for s in mine[1:]:
                for layer in range(L):
                    b.kv(s, layer, 0, before, *b.kv(mine[0], layer, 0, before))
        rows = [(prompts[i // width], before, seqs[i]) for i in range(n)]
        want = host_beams(b, L, rows, groups, width, steps, end, seqs)
        scores, ended = np.full(n, -np.inf, np.float32), np.zeros(n, np.uint8)
        scores[::width] = 0.0
        for step in range(steps):
            rows, scores, ended, parents = a.beam_step(rows, width, scores, ended, end)
            assert sorted(r[2] for r in rows) == sorted(seqs)
            assert list(parents) == want[step][0], step
            assert [r[0] for r in rows] == want[step][1], step
            assert np.max(np.abs(scores - want[step][2])) <= want[step][3], step


def test_beam_search():
    """A whole search: the prompt's own best continuations, the first of them the most likely of all that were kept."""
    with Pair("g4", 2) as (pair, a, b):
        prompt = [int(t) for t in np.random.RandomState(3).randint(0, 1000, 75)]
        found = a.beam_search(prompt, 4, 6, seqs=[3, 9, 1, 0])
        assert len(found) == 4 and all(len(t) == 6 for t, _ in found)
        assert [s for _, s in found] == sorted((s for _, s in found), reverse=True)
        for tokens, score in found:  # its log probability by single steps on the other device
            text = prompt + tokens
            total = off = 0.0
            b.rows_step([(t, i, 5) for i, t in enumerate(prompt[:-1])], logits=False)
            for i in range(len(prompt) - 1, len(text) - 1):
                x = b.step(5, text[i], i).astype(np.float64)
                total += x[text[i + 1]] - x.max() - np.log(np.sum(np.exp(x - x.max())))
                off += 2 * 4e-5 * np.max(np.abs(x))
            assert abs(total - score) <= off
        greedy = a.beam_search(prompt, 1, 6, seqs=[4])
        assert greedy[0][1] <= found[0][1] + off
        end = found[0][0][2]
        short = a.beam_search(prompt, 4, 6, end_token=end)
        assert any(t[-1] == end and len(t) <= 6 for t, _ in short)
        assert all(end not in t[:-1] for t, _ in short)


def test_refusals():
    with Pair("g4") as (pair, dev):
        for args, text in (((12, 5, [1]), "sequence 12"), ((0, 701, [1]), "positions"), ((0, 5, [0]), "itself"), ((0, 5, [1, 1]), "twice"),
                           ((0, 5, [12]), "sequence 12"), ((0, 5, [-1]), "sequence -1")):
            with pytest.raises(va.VitnaError, match=text):
                dev.kv_fork(*args)
        dev.kv_fork(0, 5, [])
        dev.kv_fork(0, 0, [1])
        ok = [(1, 5, 0), (1, 5, 1)]
        for rows, width, end, ended, text in (([(1, 5, 0), (1, 5, 0)], 2, -1, 0, "both in sequence 0"), ([(1, 700, 0), (1, 5, 1)], 2, -1, 0, "position 700"),
                                              (ok, 2, 1000, 0, "vocabulary"), (ok, 2, -1, 1, "has ended"), ([(1000, 5, 0), (1, 5, 1)], 1, -1, 0, "token 1000")):
            with pytest.raises(va.VitnaError, match=text):
                dev.beam_step(rows, width, [0.0] * 2, [ended] * 2, end)
        with pytest.raises(ValueError):
            dev.beam_step(ok, 3, [0.0] * 2, [0] * 2)
        with pytest.raises(ValueError):
            dev.beam_search([], 2, 3)
        rows, scores, _, parents = dev.beam_step(ok, 2, [-np.inf, np.nan], [0, 0])  # nothing continues
        assert list(parents) == [-1, -1] and np.all(scores == -np.inf) and sorted(r[2] for r in rows) == [0, 1]
        model = va.Model(va.shape(**dict(SPECS["g4"], attention=0)), 3)
        none = va.Device(model)
        try:
            with pytest.raises(va.VitnaError, match="no attention"):
                none.set_window(5, 1)
        finally:
            none.close()
            model.free()
