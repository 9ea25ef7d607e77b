"""Serving sequences of unequal lengths over a paged cache (trixium_b200.decoder.PagedDecoder): greedy
tokens equal the batch-1 decoder's (itself pinned to the oracle model) whatever the chunks, the slots and
the pages; sampled tokens are those of the sampler's definition on the step's logits."""
import numpy as np
import pytest
import torch

from test_sample_gpu import draw

pytestmark = pytest.mark.gpu

PROMPTS = [[5, 17, 300, 42, 999, 0, 7], [1], [640, 12, 12, 7, 800, 33, 4, 4, 90, 1, 2, 77, 650, 13, 8, 9, 10, 11, 2], [3, 2]]


def weights(name, seed=5):
    from trixium_b200 import decoder as D
    return D.SyntheticWeights(D.CONFIGS[name], seed=seed)


@pytest.mark.parametrize("name", ["tiny", "tiny-kv1", "tiny-hd256", "tiny-kseg"])
@pytest.mark.parametrize("max_rows,graph", [(64, False), (5, True)])
def test_greedy_tokens_match_decoder(name, max_rows, graph):
    from trixium_b200 import decoder as D
    w = weights(name)
    want = [D.Decoder(w, max_pos=64).generate(p, 12) for p in PROMPTS]
    pd = D.PagedDecoder(w, len(PROMPTS), max_pos=64, max_rows=max_rows)
    if graph:
        pd.capture()
    assert pd.generate(PROMPTS, 12) == want
    assert pd.plan.n_free.item() == pd.n_pages and pd.lens == [0] * len(PROMPTS)
    assert sorted(pd.free.tolist()) == list(range(pd.n_pages))
    assert pd.generate(PROMPTS[::-1], 12) == want[::-1]  # the pages come back in another order


def test_more_prompts_than_slots_and_few_pages():
    from trixium_b200 import decoder as D
    w = weights("tiny")
    prompts = PROMPTS * 2
    want = [D.Decoder(w, max_pos=64).generate(p, 6) for p in PROMPTS] * 2
    pd = D.PagedDecoder(w, 2, max_pos=32, n_pages=4, max_rows=8)
    assert pd.generate(prompts, 6) == want


def test_long_prompt_in_chunks():
    """A prompt longer than the tile sizes, in chunks that end inside pages and tiles, beside a short one."""
    from trixium_b200 import decoder as D
    w = weights("tiny")
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 1000, 330).tolist(), rng.integers(0, 1000, 21).tolist()]
    want = [D.Decoder(w, max_pos=400).generate(p, 4) for p in prompts]
    for rows in (150, 37):
        pd = D.PagedDecoder(w, 2, max_pos=400, page=32, max_rows=rows)
        assert pd.generate(prompts, 4) == want, rows


def test_sampled_tokens_are_the_definition_on_the_logits():
    from trixium_b200 import decoder as D
    pd = D.PagedDecoder(weights("tiny"), 3, max_pos=64, max_rows=32)
    cfg = [dict(temperature=0.9, top_k=50, top_p=0.9), dict(), dict(temperature=1.2, min_p=0.02)]
    for s, c in enumerate(cfg):
        pd.set_sampling(s, **c)
    tokens = [PROMPTS[0], PROMPTS[2], PROMPTS[3]]
    for step in range(5):
        pd.rand.copy_(torch.rand(3, generator=torch.Generator().manual_seed(step)))
        pd.step(tokens)
        x, u = pd.logits.double().cpu().numpy(), pd.rand.double().cpu().numpy()
        f = lambda v: float(np.float32(v))
        want = [draw(x[s], u[s], f(c.get("temperature", 0)), c.get("top_k", 0), f(c.get("top_p", 1.0)), f(c.get("min_p", 0)))
                for s, c in enumerate(cfg)]
        assert pd.tok.tolist() == want, step
        tokens = [None] * 3
    assert pd.ctx.errors() == 0
    pd.finish(range(3))
    a = pd.generate(PROMPTS, 8, sampling=[dict(temperature=1.0)] * 4, seed=1)
    assert a == pd.generate(PROMPTS, 8, sampling=[dict(temperature=1.0)] * 4, seed=1)
    assert a != pd.generate(PROMPTS, 8, sampling=[dict(temperature=1.0)] * 4, seed=2)


def test_window_and_sinks_that_cover_everything_change_nothing():
    from trixium_b200 import decoder as D
    w = weights("tiny")

    def run(**kw):
        pd = D.PagedDecoder(w, 4, max_pos=64, max_rows=64, **kw)
        return pd.generate(PROMPTS, 6), pd.logits.clone()
    full, logits = run()
    assert run(window=64)[0] == full
    assert run(window=4, sinks=64)[0] == full
    assert not torch.equal(run(window=4)[1], logits)  # (a random model's greedy tokens need not change)


def test_refusals():
    from trixium_b200 import decoder as D
    with pytest.raises(ValueError, match="DeltaNet"):
        D.PagedDecoder(weights("tiny-hybrid"), 2)
    w = weights("tiny")
    with pytest.raises(ValueError):
        D.PagedDecoder(w, 0)
    with pytest.raises(ValueError):
        D.PagedDecoder(w, 8, max_rows=4)
    pd = D.PagedDecoder(w, 2, max_pos=32, max_rows=16, n_pages=1)
    with pytest.raises(ValueError):
        pd.generate([[]], 3)
    with pytest.raises(ValueError):
        pd.step([[1] * 20, []])
    with pytest.raises(ValueError):
        pd.step([[1]])
    with pytest.raises(ValueError):
        pd.generate([[1] * 33], 1)
    with pytest.raises(ValueError, match="pass max_pos"):
        pd.generate([[1] * 14], 4)  # 17 positions, one page of 16


def test_few_pages():
    """With a page for one sequence only, prompts wait for it; a step that needs a second one is refused and
    changes nothing; capturing with every page taken works."""
    from trixium_b200 import decoder as D
    w = weights("tiny")
    want = [D.Decoder(w, max_pos=32).generate(p, 4) for p in ([1, 2], [3])]
    pd = D.PagedDecoder(w, 2, max_pos=32, max_rows=16, n_pages=1)
    assert pd.generate([[1, 2], [3]], 4) == want
    pd.step([[1, 2], []])
    with pytest.raises(ValueError, match="pool"):
        pd.step([None, [3]])
    got = [int(pd.tok[0])]
    pd.capture()
    for _ in range(3):
        pd.step([None, []])
        got.append(int(pd.tok[0]))
    assert got == want[0]
    assert pd.plan.n_free.item() == 0 and pd.lens == [5, 0]
    pd.finish([0])
    assert pd.plan.n_free.item() == 1
    pd.ctx.raise_on_error()


def test_capture_behind_other_work_keeps_the_tokens(monkeypatch):
    """Work that reaches the current stream right behind capture()'s wait for it delays nothing that the capture
    needs: the slots go on from their own last tokens."""
    from trixium_b200 import decoder as D
    w = weights("tiny")
    want = [D.Decoder(w, max_pos=64).generate(p, 4) for p in PROMPTS[:3]]
    pd = D.PagedDecoder(w, 3, max_pos=64, max_rows=32)
    pd.step(PROMPTS[:3])
    got = [pd.tok.tolist()]
    wait = torch.cuda.Stream.wait_stream

    def wait_then_busy(self, stream):
        wait(self, stream)
        torch.cuda._sleep(200_000_000)  # some 0.1 s of a plain kernel
    monkeypatch.setattr(torch.cuda.Stream, "wait_stream", wait_then_busy)
    pd.capture()
    monkeypatch.undo()
    assert pd.tok.tolist() == got[0]
    for _ in range(3):
        pd.step([None] * 3)
        got.append(pd.tok.tolist())
    assert [list(t) for t in zip(*got)] == want


@pytest.mark.parametrize("graph", [False, True])
def test_a_waiting_slot_keeps_its_token_and_logits(graph):
    """A decoding slot waits while another goes on (and a third starts and ends), then goes on from its own
    last token."""
    from trixium_b200 import decoder as D
    w = weights("tiny")
    want = [D.Decoder(w, max_pos=64).generate(p, 7) for p in PROMPTS[:2]]
    pd = D.PagedDecoder(w, 3, max_pos=64, max_rows=32)
    got = [[], []]

    def step(*tokens, took):
        pd.step(list(tokens))
        for s in took:
            got[s].append(int(pd.tok[s]))
    step(PROMPTS[0], PROMPTS[1], [], took=(0, 1))
    logits = pd.logits[1].clone()
    for third in ([], PROMPTS[2], None):
        step(None, [], third, took=(0,))
        assert int(pd.tok[1]) == got[1][-1] and torch.equal(pd.logits[1], logits)
    pd.finish([2])
    if graph:
        pd.capture()
        assert pd.tok.tolist()[:2] == [g[-1] for g in got] and torch.equal(pd.logits[1], logits)
        pd.step([[], [], PROMPTS[3]])
        step(None, None, None, took=(0, 1))
    for _ in range(2):
        step(None, None, [], took=(0, 1))
    assert got[0] == want[0][:len(got[0])] and got[1] == want[1][:len(got[1])]
    assert len(got[1]) == (4 if graph else 3)
    pd.ctx.raise_on_error()


def test_finish_takes_any_iterable():
    from trixium_b200 import decoder as D
    w = weights("tiny")
    pd = D.PagedDecoder(w, 2, max_pos=32, max_rows=16, n_pages=2)
    for slots in (iter([0, 1]), range(2), {1, 0}):
        pd.step([[1, 2], [3]])
        pd.finish(slots)
        assert pd.lens == [0, 0] == pd.plan.lens.tolist() and pd.plan.n_free.item() == 2
    assert pd.generate(PROMPTS[:1], 2) == [D.Decoder(w, max_pos=32).generate(PROMPTS[0], 2)]


@pytest.mark.parametrize("graph", [False, True])
def test_steps_draw_a_number_each(graph):
    """Without numbers from the caller every step draws its own, the same ones again from the same seed, and the
    tokens spread; a number that the caller wrote stays in use until it is taken back."""
    from trixium_b200 import decoder as D
    w = weights("tiny")

    def run(seed):
        pd = D.PagedDecoder(w, 3, max_pos=64, max_rows=16, seed=seed)
        pd.set_sampling(0, temperature=1e4)  # near enough even over the vocabulary
        pd.set_sampling(1, temperature=1e4)
        pd.rand[1] = 0.5
        pd.step([[1], [2], [3]])
        if graph:
            pd.capture()
        toks = []
        for _ in range(24):
            pd.step([None] * 3)
            toks.append(pd.tok.tolist())
        pd.ctx.raise_on_error()
        return np.array(toks), pd
    a, pd = run(7)
    V = pd.cfg.vocab
    # 24 even draws of V tokens fall into both halves but for 2 in 2^24, and the same token twice in a row
    # all along never; u = 1/2 of nearly even weights is near the middle.
    assert 0 < (a[:, 0] < V // 2).sum() < 24 and len(set(a[:, 0])) > 4
    assert (abs(a[:, 1] - V / 2) < V / 20).all()
    b, _ = run(7)
    assert (a == b).all()
    assert (run(8)[0][:, 0] != a[:, 0]).any()
    pd.rand[1] = float("nan")
    later = []
    for _ in range(24):
        pd.step([None] * 3)
        later.append(int(pd.tok[1]))
    assert 0 < sum(t < V // 2 for t in later) < 24


def test_an_empty_slot_has_no_last_token():
    """None for a slot that holds no sequence is refused (its token is that of the one before), eager and captured,
    and changes nothing."""
    from trixium_b200 import decoder as D
    pd = D.PagedDecoder(weights("tiny"), 2, max_pos=32, max_rows=16)
    with pytest.raises(ValueError, match="empty slot"):
        pd.step([None, [1]])
    pd.step([[1, 2], [3]])
    pd.capture()
    pd.step([None, None])
    pd.finish([1])
    with pytest.raises(ValueError, match="empty slot"):
        pd.step([None, None])
    assert pd.lens == [3, 0] == pd.plan.lens.tolist()
    pd.step([None, [5]])
    pd.step([None, None])
    assert pd.lens == [5, 2] == pd.plan.lens.tolist() and pd.ctx.errors() == 0


def test_settings_for_fewer_prompts_are_refused():
    """Before anything runs: the slots stay empty and the next call works."""
    from trixium_b200 import decoder as D
    w = weights("tiny")
    pd = D.PagedDecoder(w, 2, max_pos=32, max_rows=16)
    with pytest.raises(ValueError, match="sampling has 2 entries for 4 prompts"):
        pd.generate(PROMPTS, 3, sampling=[None, dict(temperature=1.0)])
    assert pd.lens == [0, 0]
    assert pd.generate(PROMPTS[:2], 3, sampling=[None, None]) == [D.Decoder(w, max_pos=32).generate(p, 3) for p in PROMPTS[:2]]


@pytest.mark.parametrize("bad", ["x", 2 ** 40, None])
def test_a_step_of_no_tokens_changes_nothing(bad):
    """Tokens that are no 32-bit integers raise before anything is done."""
    from trixium_b200 import decoder as D
    w = weights("tiny")
    pd = D.PagedDecoder(w, 2, max_pos=32, max_rows=16)
    with pytest.raises((ValueError, TypeError, RuntimeError)):
        pd.step([[1, bad], [2]])
    assert pd.lens == [0, 0] == pd.plan.lens.tolist()
    assert pd.generate(PROMPTS[:1], 2) == [D.Decoder(w, max_pos=32).generate(PROMPTS[0], 2)]
