"""Drafted trees and bounded caches through the engine, the generation loop and the command line, against the plain models."""
import random
import subprocess
import sys

import numpy as np
import pytest
import torch

from helpers import BF16_REL, FP32_REL, TINY, assert_close, make_folder, prompts_for
from plain.evicting import PlainEvicting
from plain.model import PlainQwen3
from test_gpu_engine import ROOT

pytestmark = pytest.mark.gpu

CASES = [("A", "float32"), ("B", "float32"), ("D", "float32"), ("A", "bfloat16"), ("D", "bfloat16")]


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("models")
    return {(n, d): make_folder(root, n, torch.float32 if d == "float32" else torch.bfloat16) for n, d in CASES + [("C", "float32"), ("B", "bfloat16")]}


def _engine(folder, dtype, max_tokens=2048, **kw):
    from mynah_slm_b200.engine.engine import Engine
    return Engine.from_folder(folder, dtype=dtype, max_tokens=max_tokens, **kw)


def _prompt_step(eng, prompts):
    from mynah_slm_b200.engine.engine import StepEntry
    slots = [eng.open_sequence() for _ in prompts]
    eng.step([StepEntry(s, p, ()) for s, p in zip(slots, prompts)])
    return slots


def _random_tree(rng, n, vocab):
    parents = [-1] + [max(0, i - 1 - int(rng.random() ** 2 * 4)) for i in range(1, n)]
    return [rng.randrange(vocab) for _ in range(n)], parents


def _path(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out[::-1]


@pytest.mark.parametrize("name,dtype", CASES, ids=[f"{n}-{d}" for n, d in CASES])
def test_every_row_of_a_tree_has_the_logits_of_its_path(folders, name, dtype):
    from mynah_slm_b200.engine.engine import StepEntry, TreeEntry
    plain = PlainQwen3.from_folder(folders[(name, dtype)])
    eng = _engine(folders[(name, dtype)], dtype)
    tol = FP32_REL if dtype == "float32" else BF16_REL
    rng = random.Random(3)
    vocab = TINY[name]["vocab_size"]
    prompts = [list(p) for p in prompts_for(name, [5, 70, 63])]
    slots = _prompt_step(eng, prompts)
    for sizes in ((1, 12, 3), (20, 1, 70)):
        trees = [_random_tree(rng, n, vocab) for n in sizes]
        seen = {}

        def choose(logits):
            seen["logits"] = logits.cpu().numpy()
            # a walk down some branch of every tree: what follows a row is its last child's token where it has one
            pick, at = [], 0
            for tokens, parents in trees:
                kids = {p: i for i, p in enumerate(parents) if p >= 0}
                pick += [tokens[kids[i]] if i in kids else int(np.argmax(seen["logits"][at + i])) for i in range(len(tokens))]
                at += len(tokens)
            return torch.tensor(pick, dtype=torch.int32, device=logits.device)
        before = [eng.length(s) for s in slots]
        got = eng.step_tree([TreeEntry(s, *t) for s, t in zip(slots, trees)], choose)
        at = 0
        for b, (tokens, parents) in enumerate(trees):
            want = np.stack([plain.forward(prompts[b] + [tokens[j] for j in _path(parents, i)])[-1] for i in range(len(tokens))])
            assert_close(want, seen["logits"][at:at + len(tokens)], tol, f"tree {b}")
            kids = {}
            for i, p in enumerate(parents):
                kids.setdefault(p, []).append(i)
            walk = [0]
            while walk[-1] in kids:                        # the lowest child with the chosen token
                last = kids[walk[-1]][-1]
                walk.append(next(c for c in kids[walk[-1]] if tokens[c] == tokens[last]))
            assert got[b].tokens == [tokens[i] for i in walk[1:]]
            assert eng.length(slots[b]) == before[b] + len(walk)
            prompts[b] += [tokens[i] for i in walk]
            at += len(tokens)
        # the accepted rows are where a sequence that had taken them one by one would have them
        nxt = [r.next for r in got]
        logits = eng.step([StepEntry(s, (t,), (0,)) for s, t in zip(slots, nxt)]).cpu().numpy()
        for b in range(3):
            prompts[b].append(nxt[b])
            assert_close(plain.forward(prompts[b])[-1][None], logits[b][None], tol, f"after the tree, {b}")
    eng.check_status()


@pytest.mark.parametrize("name", ["A", "D"])
def test_drafted_generation_is_greedy_generation(folders, name):
    from mynah_slm_b200 import LLM
    llm = LLM(folders[(name, "float32")], dtype="float32", max_tokens=4096)
    rng = random.Random(5)
    base = [rng.randrange(100) for _ in range(9)]
    prompts = [base * 4, base[:5] * 3 + [1], [7], [rng.randrange(100) for _ in range(70)]]
    want = [(r.tokens, r.finish_reason, r.produced) for r in llm.generate(prompts, max_new=40, temp=0.0)]
    free = llm.engine.free_tokens()
    for draft in (1, 4, 30, 90):
        got = llm.generate(prompts, max_new=40, temp=0.0, draft=draft, max_batch=3)
        assert [(r.tokens, r.finish_reason, r.produced) for r in got] == want
        assert llm.engine.free_tokens() == free
    # up to the model's last position
    long = [i % 5 for i in range(TINY[name]["max_position_embeddings"] - 6)]
    a, b = (llm.generate([long], max_new=50, temp=0.0, ignore_eos=True, draft=d)[0] for d in (0, 12))
    assert (a.tokens, a.finish_reason) == (b.tokens, b.finish_reason) and a.finish_reason == "context"


def test_drafted_steps_gain_tokens(folders):
    """A model that says what its text says next takes several tokens a step."""
    from mynah_slm_b200 import LLM
    llm = LLM(folders[("D", "bfloat16")], dtype="bfloat16", max_tokens=4096)
    out = llm.generate([[3, 4]], max_new=200, temp=0.0, ignore_eos=True)[0]
    eng = llm.engine
    steps = {"n": 0}
    real = eng.step_tree

    def counted(*a, **k):
        steps["n"] += 1
        return real(*a, **k)
    eng.step_tree = counted
    again = llm.generate([[3, 4] + out.tokens[:150]], max_new=50, temp=0.0, ignore_eos=True, draft=8)[0]
    assert again.produced == 50 and steps["n"] <= 49


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_text_that_repeats_is_generated_in_fewer_steps(folders, dtype):
    """A model whose next token goes by the last one alone (its layers add nothing) soon repeats itself: its drafts are accepted."""
    from mynah_slm_b200 import LLM
    llm = LLM(folders[("B", dtype)], dtype=dtype, max_tokens=4096)
    for layer in llm.engine.model.layers:
        layer.mixer.w_o.zero_()
        layer.ffn.w_down.zero_()
    text = [3] + llm.generate([[3]], max_new=400, temp=0.0, ignore_eos=True)[0].tokens
    start = text.index(text[-1])                           # from here on the text goes round
    period = text.index(text[-1], start + 1) - start
    assert start + 3 * period < 300 and all(text[i] == text[i + period] for i in range(start, len(text) - period))
    at = start + 2 * period + 1
    results, real = [], llm.engine.step_tree

    def counted(entries, *a, **k):
        out = real(entries, *a, **k)
        results.extend(out)
        return out
    llm.engine.step_tree = counted
    got = llm.generate([text[:at]], max_new=60, temp=0.0, ignore_eos=True, draft=8)[0]
    assert got.tokens == text[at:at + 60]
    # the round is known when the first tree is drafted: its last place gives min(8, period) tokens, and all of them are right
    gain = 1 + min(8, period)
    assert sum(len(r.tokens) + 1 for r in results) == 59 and len(results) <= -(-59 // gain) + 1
    assert max(len(r.tokens) for r in results) >= min(8, period)


def test_what_cannot_draft_refuses(folders):
    from mynah_slm_b200 import LLM
    from mynah_slm_b200.engine.engine import EngineError, KeepRows, TreeEntry
    from mynah_slm_b200.engine.generate import GenerationError
    llm = LLM(folders[("A", "float32")], dtype="float32", max_tokens=256)
    with pytest.raises(GenerationError):
        llm.generate([[1]], temp=0.5, draft=4)
    with pytest.raises(GenerationError):
        llm.generate([[1]], temp=0.0, repeat_penalty=1.1, draft=4)
    with pytest.raises(GenerationError):
        llm.generate([[1]], temp=0.0, draft=-1)
    eng = llm.engine
    s = eng.open_sequence()
    for tokens, parents in (([1, 2], [-1, 1]), ([1, 2], [0, 0]), ([1], []), ([], []), ([1, 10 ** 6], [-1, 0]), ([1, 2], [-1, -1])):
        with pytest.raises(EngineError):
            eng.step_tree([TreeEntry(s, tokens, parents)])
    with pytest.raises(EngineError):
        eng.step_tree([TreeEntry(s, [1], [-1]), TreeEntry(s, [1], [-1])])
    with pytest.raises(EngineError):
        eng.step_tree([TreeEntry(s, [1, 2], [-1, 0])], choose=lambda logits: torch.zeros(2, dtype=torch.int64, device=logits.device))
    windowed = _engine(folders[("C", "float32")], "float32", 256)
    t = windowed.open_sequence()
    with pytest.raises(EngineError):
        windowed.step_tree([TreeEntry(t, [1], [-1])])
    with pytest.raises(EngineError):
        _engine(folders[("C", "float32")], "float32", 256, keep=KeepRows(64, 32, 8))
    for bad in ((10, 20, 2, 2), (10, 8, 9, 0), (10, 0, 0, 0), (10, 8, -1, 2)):
        with pytest.raises(EngineError):
            KeepRows(*bad)
    bounded = _engine(folders[("A", "float32")], "float32", 256, keep=KeepRows(64, 32, 8))
    b = bounded.open_sequence()
    with pytest.raises(EngineError):
        bounded.step_tree([TreeEntry(b, [1], [-1])])
    with pytest.raises(EngineError):
        bounded.decode_loop([b], [1], 2)


# -------------------------------------------------------------- bounded caches

@pytest.mark.parametrize("name", ["A", "B", "D"])
@pytest.mark.parametrize("graphs", [True, False], ids=["graphs", "eager"])
def test_a_bounded_cache_is_the_plain_one(folders, name, graphs):
    from mynah_slm_b200.engine.engine import KeepRows, StepEntry
    keep = KeepRows(40, 24, 9, 3)
    eng = _engine(folders[(name, "float32")], "float32", 1024, keep=keep, use_graphs=graphs)
    plain = [PlainEvicting.from_folder(folders[(name, "float32")]) for _ in range(2)]
    prompts = [list(p) for p in prompts_for(name, [90, 17])]
    for p in plain:
        p.start(40, 24, 9, 3)
    slots = [eng.open_sequence() for _ in prompts]
    got = eng.step([StepEntry(s, p, (len(p) - 1,)) for s, p in zip(slots, prompts)]).cpu().numpy()
    want = np.stack([m.step(p)[-1] for m, p in zip(plain, prompts)])
    assert_close(want, got, FP32_REL, "prompts")
    rng = random.Random(1)
    for i in range(60):                                    # several evictions of each
        toks = [rng.randrange(TINY[name]["vocab_size"]) for _ in slots]
        got = eng.step([StepEntry(s, (t,), (0,)) for s, t in zip(slots, toks)]).cpu().numpy()
        want = np.stack([m.step([t])[-1] for m, t in zip(plain, toks)])
        assert_close(want, got, FP32_REL, f"step {i}")
        for s, m in zip(slots, plain):
            assert eng.length(s) == len(m.held[0][0]["m"]) <= 40 and eng.positions(s) == m.pos
    piece = [rng.randrange(TINY[name]["vocab_size"]) for _ in range(30)]
    got = eng.step([StepEntry(slots[1], piece, range(30))]).cpu().numpy()      # a further piece of a prompt
    assert_close(plain[1].step(piece), got, FP32_REL, "piece")
    eng.check_status()
    # the sums are the plain ones too
    g = eng.cache.views[0].group
    for l in range(plain[0].L):
        pages = torch.tensor(eng.cache.pages.held(slots[0], g)[0], device=eng.device)
        n = eng.length(slots[0])
        m = eng.cache.views[l].mass[pages].permute(1, 0, 2).reshape(plain[0].KV, -1)[:, :n].double().cpu().numpy()
        assert np.allclose(m, np.stack([c["m"] for c in plain[0].held[l]]), rtol=1e-3, atol=1e-4)


def test_a_bound_that_is_never_reached_changes_nothing(folders):
    from mynah_slm_b200.engine.engine import KeepRows, StepEntry
    for name, dtype in (("B", "float32"), ("D", "bfloat16")):
        plain = PlainQwen3.from_folder(folders[(name, dtype)])
        eng = _engine(folders[(name, dtype)], dtype, 1024, keep=KeepRows(400, 300, 50))
        p = list(prompts_for(name, [70])[0])
        s = eng.open_sequence()
        logits = eng.step([StepEntry(s, p[:40], (39,))]).cpu().numpy()
        tol = FP32_REL if dtype == "float32" else BF16_REL
        assert_close(plain.forward(p[:40])[-1][None], logits, tol)
        for i in range(40, 70):
            logits = eng.step([StepEntry(s, (p[i],), (0,))]).cpu().numpy()
            assert_close(plain.forward(p[:i + 1])[-1][None], logits, tol)


@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("D", "bfloat16")])
def test_generation_over_a_bounded_cache(folders, name, dtype):
    """More tokens than the cache has rows for; the same tokens whatever the batch and with slots that are used again."""
    from mynah_slm_b200 import LLM
    from mynah_slm_b200.engine.engine import KeepRows
    n = TINY[name]["max_position_embeddings"]
    llm = LLM(folders[(name, dtype)], dtype=dtype, max_tokens=3 * 64, keep=KeepRows(60, 40, 12))
    prompts = [[1, 2, 3], [5] * 20, [9, 8, 7, 6], [4]]
    out = llm.generate(prompts, max_new=150, temp=0.0, ignore_eos=True)
    assert all(len(r.tokens) == 150 and r.finish_reason == "length" for r in out)
    llm.engine.check_status()
    assert llm.engine.free_tokens() == 3 * 64
    if dtype == "float32":
        alone = [llm.generate([p], max_new=150, temp=0.0, ignore_eos=True)[0].tokens for p in prompts]
        assert alone == [r.tokens for r in out]
    end = llm.generate([[1, 2]], max_new=10 * n, temp=0.0, ignore_eos=True)[0]
    assert end.finish_reason == "context" and len(end.tokens) == n - 2 + 1


@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("B", "float32"), ("D", "float32"), ("A", "bfloat16")])
def test_a_bounded_sequence_keeps_the_same_rows_alone_and_in_a_batch(folders, name, dtype):
    """Token by token, with evictions: logits, sums and the keys that stay have the same bits alone and beside longer sequences (in 32
    bits, and with heads that the tensor cores do not take)."""
    from mynah_slm_b200.engine.engine import KeepRows, StepEntry
    rng = random.Random(9)
    vocab, n = TINY[name]["vocab_size"], 150
    text = [rng.randrange(vocab) for _ in range(n)]
    others = [[rng.randrange(vocab) for _ in range(n)] for _ in range(4)]

    def run(beside):
        eng = _engine(folders[(name, dtype)], dtype, 4096, keep=KeepRows(70, 50, 16))
        slots = [eng.open_sequence() for _ in range(1 + beside)]
        for s, o in zip(slots[1:], others):
            eng.step([StepEntry(s, o[:65], ())])               # further on than the first, so that they are cut at other steps
        logits = []
        for i in range(n):
            out = eng.step([StepEntry(s, (t[i],), (0,)) for s, t in zip(slots, [text] + others)])
            logits.append(out[0].clone())
        eng.check_status()
        held = eng.length(slots[0])
        views = []
        for view in eng.cache.views:
            pages = torch.tensor(eng.cache.pages.held(slots[0], view.group)[0], device=eng.device)
            for t in (view.mass, view.k, view.v):
                views.append(t[pages].transpose(0, 1).flatten(1, 2)[:, :held].clone())
        return torch.stack(logits), views, held
    want = run(0)
    for beside in (1, 4):
        got = run(beside)
        assert got[2] == want[2] and torch.equal(got[0], want[0])
        assert all(torch.equal(a, b) for a, b in zip(got[1], want[1]))


def test_the_command_line_drafts_and_keeps(folders):
    def run(*extra):
        cmd = [sys.executable, "-m", "mynah_slm_b200.cli", "run", "-m", folders[("A", "float32")], "--dtype", "float32", "--tokens", "1,2,3,1,2,3,1,2",
               "-n", "30", "--temp", "0", "--ignore-eos", "--no-stream", "--quiet", *extra]
        r = subprocess.run(cmd, capture_output=True, text=True, cwd=ROOT, timeout=300)
        assert r.returncode == 0, r.stderr
        return r.stdout.split()
    plain = run()
    assert run("--draft", "6") == plain and len(plain) == 30
    assert len(run("--keep", "20")) == 30
