"""Forked sessions: windows of a fork equal those of a session that prefilled the whole context itself, pages are shared
and come back, and batched windows of forks read the shared pages once with the same results."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from test_llama_gpu import make_engine, rel, small_geo  # noqa: E402


def prefill(e, session, tokens, chunk=32):
    at = 0
    while at < len(tokens):
        w = tokens[at:at + chunk]
        e.run_window(session, at, tokens=w)
        e.commit(session, len(w))
        at += len(w)


@pytest.mark.parametrize("length", [0, 1, 63, 64, 65, 150, 192])
def test_a_fork_continues_as_its_parent_would(ctx, length):
    geo = small_geo("q4_k", n_heads=4, n_kv_heads=2, hidden=512)
    e = make_engine(ctx, geo, max_context=320, max_window=32, sessions=4)
    ref = make_engine(ctx, geo, max_context=320, max_window=32, sessions=1)
    rng = np.random.default_rng(length)
    prompt = rng.integers(0, geo.vocab, length).astype(np.int32)
    e.open_session(1)
    prefill(e, 1, prompt)
    e.fork_session(1, 2)
    e.fork_session(2, 3)  # a fork of a fork
    assert e.position(2) == e.position(3) == length
    more = {s: rng.integers(0, geo.vocab, 70).astype(np.int32) for s in (1, 2, 3)}
    got = {s: [] for s in more}
    for k in range(0, 70, 7):  # interleaved: nobody writes where another reads
        for s in more:
            got[s].append(e.run_window(s, length + k, tokens=more[s][k:k + 7]))
            e.commit(s, 7)
    for s in more:
        ref.open_session(9)
        prefill(ref, 9, prompt)
        for k in range(0, 70, 7):
            want = ref.run_window(9, length + k, tokens=more[s][k:k + 7])
            np.testing.assert_array_equal(got[s][k // 7], want)
            ref.commit(9, 7)
        ref.close_session(9)
    e.close()
    ref.close()


def test_pages_live_until_their_last_session_closes(ctx):
    geo = small_geo("q8_0")
    e = make_engine(ctx, geo, max_context=128, max_window=16, sessions=3)
    prompt = np.arange(100, dtype=np.int32)
    e.open_session(1)
    prefill(e, 1, prompt, 16)
    before = e.run_window(1, 100, tokens=[5, 6, 7])
    e.abort(1)
    for turn in range(5):  # more sessions than pages, were any of them lost
        e.fork_session(1, 2)
        e.fork_session(2, 3)
        e.close_session(1)
        e.close_session(3)
        e.open_session(7)  # takes the freed pages: the survivor's context is not touched
        prefill(e, 7, prompt[::-1].copy(), 16)
        np.testing.assert_array_equal(e.run_window(2, 100, tokens=[5, 6, 7]), before)
        e.abort(2)
        e.close_session(7)
        e.fork_session(2, 1)
        e.close_session(2)
    e.close()


def test_fork_refusals(ctx):
    from clusterlm_b200 import ClmError

    geo = small_geo("q8_0")
    e = make_engine(ctx, geo, max_context=128, max_window=16, sessions=2)
    with pytest.raises(ClmError) as ex:
        e.fork_session(1, 2)
    assert ex.value.name == "kNotFound"
    e.open_session(1)
    with pytest.raises(ClmError) as ex:
        e.fork_session(1, 1)
    assert ex.value.name == "kAlreadyExists"
    e.run_window(1, 0, tokens=[1, 2])
    with pytest.raises(ClmError) as ex:
        e.fork_session(1, 2)
    assert ex.value.name == "kFailedPrecondition"
    e.commit(1, 2)
    e.fork_session(1, 2)
    with pytest.raises(ClmError) as ex:
        e.fork_session(1, 3)
    assert ex.value.name == "kResourceExhausted"
    e.close()


@pytest.mark.parametrize("length,q,tree", [(200, 8, False), (200, 16, True), (130, 5, False), (40, 8, False)])
def test_batched_windows_of_forks(ctx, oracle, length, q, tree):
    """Four forks and an unrelated session in one window: each session's logits equal its own window's (single sessions
    read their pages alone) within the operands' rounding, eagerly, captured and replayed."""
    from test_llama_gpu import _tree16

    geo = small_geo("q8_0", n_heads=8, n_kv_heads=2, hidden=1024)
    e = make_engine(ctx, geo, max_context=512, max_window=96, sessions=5)
    rng = np.random.default_rng(3)
    e.open_session(1)
    prefill(e, 1, rng.integers(0, geo.vocab, length).astype(np.int32))
    for s in (2, 3, 4):
        e.fork_session(1, s)
    e.open_session(5)
    prefill(e, 5, rng.integers(0, geo.vocab, 90).astype(np.int32))
    for s, own in ((1, 9), (2, 1), (3, 75)):  # histories of their own
        w = rng.integers(0, geo.vocab, own).astype(np.int32)
        e.run_window(s, length, tokens=w)
        e.commit(s, own)
    order = [1, 2, 3, 4, 5]
    parents = _tree16() if tree else None
    for _ in range(4):  # eager, captured, replayed, replayed
        pos = [e.position(s) for s in order]
        toks = rng.integers(0, geo.vocab, (5, q)).astype(np.int32)
        got = e.run_batch_window(order, pos, toks, parents)
        for s in order:
            e.abort(s)
        for i, s in enumerate(order):
            alone = (e.run_tree_window(s, pos[i], parents, tokens=toks[i]) if tree
                     else e.run_window(s, pos[i], tokens=toks[i]))
            assert rel(got[i], alone) < 2e-2, (s, rel(got[i], alone))
            if tree:
                e.commit_path(s, [0])
            else:
                e.commit(s, 3)
    e.close()


def test_forked_rounds_follow_the_parent_and_part_by_seed(ctx):
    geo = small_geo("q4_k")
    e = make_engine(ctx, geo, max_context=256, max_window=16, sessions=3)
    prompt = np.random.default_rng(8).integers(0, geo.vocab, 70).astype(np.int32)
    e.open_session(1)
    e.spec_begin(1, prompt, 4, temperature=1.0, seed=5)
    e.fork_session(1, 2)
    e.fork_session(1, 3)
    a, b, c = ([int(t) for _ in range(12) for t in e.spec_round(s, 4, temperature=1.0, seed=seed)]
               for s, seed in ((1, 5), (2, 5), (3, 6)))
    assert a == b and a != c
    e.close()


@pytest.mark.parametrize("length", [64, 100])
def test_forks_of_a_split_model_equal_the_whole_ones(ctx, length):
    """Prefix, middle and tail (with its draft head) each fork: their windows chained are the whole engine's, to the bit."""
    from clusterlm_b200.engine import ROLE_MIDDLE, ROLE_PREFIX, ROLE_TAIL

    geo = small_geo(n_layers=3)
    kw = dict(max_context=192, max_window=16, sessions=3)
    whole = make_engine(ctx, geo, **kw)
    stages = [make_engine(ctx, geo, ROLE_PREFIX, 0, 1, **kw), make_engine(ctx, geo, ROLE_MIDDLE, 1, 2, **kw),
              make_engine(ctx, geo, ROLE_TAIL, 2, 3, **kw)]
    rng = np.random.default_rng(length)
    prompt = rng.integers(0, geo.vocab, length).astype(np.int32)

    def window(s, at, toks, keep):
        want = whole.run_window(s, at, tokens=toks)
        rec = stages[0].run_window(s, at, tokens=toks)
        rec = stages[1].run_window(s, at, records=rec)
        np.testing.assert_array_equal(stages[2].run_window(s, at, records=rec), want)
        for e in (whole, *stages):
            e.commit(s, keep)

    for e in (whole, *stages):
        e.open_session(1)
    for at in range(0, length, 16):
        window(1, at, prompt[at:at + 16], len(prompt[at:at + 16]))
    for e in (whole, *stages):
        e.fork_session(1, 2)
        e.fork_session(2, 3)
        assert [e.position(s) for s in (1, 2, 3)] == [length] * 3
    at = {s: length for s in (1, 2, 3)}
    for q, keep in [(4, 4), (8, 3), (4, 1), (16, 16)]:
        for s in (2, 1, 3):
            window(s, at[s], rng.integers(0, geo.vocab, q).astype(np.int32), keep)
            at[s] += keep
    drafts = [e.mtp_draft(5, 3) for e in (whole, stages[2])]
    np.testing.assert_array_equal(*drafts)
    for e in (whole, *stages):
        e.close_session(1)
        e.fork_session(3, 1)  # the place and the pages go round
        assert e.position(1) == at[3]
    at[1] = at[3]
    window(1, at[1], rng.integers(0, geo.vocab, 4).astype(np.int32), 4)
    for e in (whole, *stages):
        e.close()
