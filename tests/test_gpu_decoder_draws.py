"""GPU tests of BitLlamaHip's sampled picks used together: the host's pick (sample) between
the device loop's captured steps."""
import numpy as np
import pytest
import torch

import serve_ref as ref
from test_gpu_model import gpu_model
from test_gpu_serve import host
from test_model_oracle import TinyCfg, tiny_weights

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

F = dict(temperature=0.9, top_k=12, top_p=0.9, min_p=0.01)
PROMPT = [3, 9, 27, 5]


def model_of(seed=3):
    cfg = TinyCfg()
    return cfg, gpu_model(cfg, tiny_weights(cfg, seed), max_rows=8)


def picked(logits, u, f=F):
    return ref.sample_one(logits, f["temperature"], f["top_k"], f["top_p"], f["min_p"], float(u))[0]


def definition(cfg, tokens, u, first, n, f=F, seed=3):
    """The picks after `tokens`, of a model of its own: its first is drawn with u[first]."""
    _, m = model_of(seed)
    logits = host(m.prefill(tokens)).copy()
    got = []
    for i in range(n):
        got.append(picked(logits, u[first + i], f))
        logits = host(m.forward_one(got[-1])).copy()
    return got


def test_a_captured_steps_buffers_stay_where_they_are():
    """sample() of other filters between replays: the captured step goes on by its own filters and
    numbers, and writes nothing into memory that was taken meanwhile."""
    cfg, m = model_of()
    u = np.random.default_rng(4).random(40).astype(np.float32)
    n = 10
    first = m.generate(PROMPT, n, u=u, **F)
    assert m.graph is not None
    held = {k: t.data_ptr() for k, t in m._loop.items() if torch.is_tensor(t)}
    m._loop["u"][m.pos:m.pos + 20].copy_(torch.from_numpy(u[n:n + 20]))
    got, tokens = [], list(PROMPT) + [int(t) for t in first]
    for step in range(4):
        # a pick by other filters: the logits are those of the last token's predecessor
        for v in (0.1, 0.9):
            m.sample(v, temperature=1.3, top_k=3)
        # whatever could have been freed is taken and marked
        taken = [torch.full((k,), 123.0, device="cuda") for k in (1, 1, 1, 1, 1, cfg.max_seq, 4096, 65536)]
        m.next_id.fill_(tokens[-1])
        m.graph.replay()
        m.pos += 1
        torch.cuda.synchronize()
        tokens.append(int(m.next_id))
        got.append(tokens[-1])
        assert all(bool((t == 123.0).all()) for t in taken)
    assert {k: t.data_ptr() for k, t in m._loop.items() if torch.is_tensor(t)} == held
    assert got == definition(cfg, list(PROMPT) + [int(t) for t in first], u, n, 4)
    # generate again, captured over the same buffers
    assert np.array_equal(m.generate(PROMPT, n, u=u, **F), first)


@pytest.mark.parametrize("use_graph", [True, False])
def test_steps_past_the_numbers_are_refused(use_graph):
    """Numbers that generate() was given beyond its tokens serve the steps after it; past them a
    step is refused and nothing moves; start_decode makes the loop greedy."""
    cfg, m = model_of()
    u = np.random.default_rng(5).random(30).astype(np.float32)
    exp = m.generate(PROMPT, 14, use_graph=use_graph, u=u[:14], **F)
    n = 9
    got = m.generate(PROMPT, n, use_graph=use_graph, u=u[:14], **F)
    assert np.array_equal(got, exp[:n])
    m.decode_steps(2, use_graph=use_graph)
    m.decode_steps(3, use_graph=use_graph)
    start = len(PROMPT)
    assert np.array_equal(m.log[start:start + 14].cpu().numpy(), exp)
    for steps in (1, 7):
        with pytest.raises(ValueError):
            m.decode_steps(steps, use_graph=use_graph)
    m.decode_steps(0, use_graph=use_graph)
    assert m.pos == start + 13 and int(m.d_pos) == m.pos and int(m.next_id) == exp[-1]
    # from here on greedily
    logits = host(m.forward_one(int(exp[-1]))).copy()
    m.greedy()
    m.start_decode()
    m.decode_steps(5, use_graph=use_graph)
    tokens, greedy = list(PROMPT) + [int(t) for t in exp], []
    for _ in range(6):
        greedy.append(int(np.flatnonzero(logits == logits.max())[-1]))
        tokens.append(greedy[-1])
        fresh = model_of()[1]
        logits = host(fresh.prefill(tokens)).copy()
    assert m.log[m.pos - 5:m.pos + 1].cpu().numpy().tolist() == greedy
    # exactly as many numbers as tokens: none is left for a step after them
    m.generate(PROMPT, 3, use_graph=use_graph, u=u[:3], **F)
    with pytest.raises(ValueError):
        m.decode_steps(1, use_graph=use_graph)
    # a single token is picked by the host alone; the loop goes on by the numbers behind it
    one = m.generate(PROMPT, 1, use_graph=use_graph, u=u[:5], **F)
    assert np.array_equal(one, exp[:1])
    m.decode_steps(4, use_graph=use_graph)
    assert np.array_equal(m.log[start:start + 5].cpu().numpy(), exp[:5])


def test_numbers_to_the_end_of_the_cache():
    cfg, m = model_of()
    u = np.random.default_rng(6).random(cfg.max_seq + 50).astype(np.float32)
    most = cfg.max_seq - len(PROMPT) + 1  # the last token needs no place
    got = m.generate(PROMPT, most, u=u, **F)
    assert got.tolist() == definition(cfg, PROMPT, u, 0, 3) + got.tolist()[3:]
    assert np.array_equal(m.generate(PROMPT, most, use_graph=False, u=u[:most], **F), got)
    with pytest.raises(ValueError):
        m.decode_steps(1)
    with pytest.raises(ValueError):
        m.generate(PROMPT, most + 1, u=u, **F)


def test_a_captured_step_replayed_past_the_caches_end():
    """Every index of a sampled step stays inside its array: steps past the last row store nothing
    and leave the log as it is, as the greedy step's do."""
    cfg, m = model_of()
    u = np.random.default_rng(7).random(cfg.max_seq).astype(np.float32)
    most = cfg.max_seq - len(PROMPT) + 1
    for sampled in (False, True):
        m.generate(PROMPT, most, **(dict(u=u, **F) if sampled else {}))
        assert m.pos == cfg.max_seq == int(m.d_pos)
        log = m.log.clone()
        caches = [t.clone() for c in m.caches for t in (c.k, c.v, c.k_scale, c.v_scale)]
        for i in range(3):
            m.graph.replay()
            torch.cuda.synchronize()
            assert int(m.d_pos) == cfg.max_seq + 1 + i
        assert torch.equal(m.log, log) and m.log.numel() == cfg.max_seq + 1
        for a, b in zip(caches, (t for c in m.caches for t in (c.k, c.v, c.k_scale, c.v_scale))):
            assert torch.equal(a, b)
    # and the model goes on as ever
    assert np.array_equal(m.generate(PROMPT, most, u=u, **F), m.generate(PROMPT, most, use_graph=False, u=u, **F))
