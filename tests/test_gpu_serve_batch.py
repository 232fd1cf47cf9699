"""The batched serving example against the single-sequence model on the tiny
Llama config: the same prompts, tokens forced to the batch's own choices.

int8 pages round each K and V value to 1 / 254 of its token's largest, about
0.7 % rms of a value; probabilities average V's part down and the residual
stream carries the rest of the layer, so the logits agree to 2e-2."""
import os
import sys

import numpy as np
import pytest

from lumina_b200 import synthetic

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples"))
TOL = 2e-2
CFG = synthetic.TINY


@pytest.fixture(scope="module")
def served(tiny_file):
    import serve_batch as sb
    model = sb.BatchModel(tiny_file, CFG["num_attention_heads"], CFG["num_key_value_heads"], CFG["rope_theta"], n_pages=80)
    rng = np.random.default_rng(3)
    allowed = rng.random(CFG["vocab_size"]) < 0.5
    prompts = [rng.integers(0, CFG["vocab_size"], n).tolist() for n in (5, 150, 33, 64, 17, 1)]
    reqs = [sb.Request(p, max_tokens=6 + i) for i, p in enumerate(prompts)]
    reqs[1].repeat_penalty, reqs[1].frequency, reqs[1].presence = 1.2, 0.01, 0.02
    reqs[2].allowed = allowed
    reqs[3].bias = {7: 100.0}
    steps = []  # logits as they left the model, the requests that get a token from them
    pick = model.pick

    def keep(logits, giving):
        steps.append((logits.cpu().numpy(), [(reqs.index(r), len(r.out)) for r in giving]))
        return pick(logits, giving)

    model.pick = keep
    outs = model.serve(reqs)
    return model, reqs, outs, steps


def test_requests_end_and_pages_return(served):
    model, reqs, outs, steps = served
    assert [len(o) for o in outs] == [r.max_tokens for r in reqs]
    assert sorted(model.free) == list(range(80))
    assert any(len(who) > 1 for _, who in steps)
    assert all(reqs[2].allowed[t] for t in outs[2])
    assert outs[3] == [7] * reqs[3].max_tokens


def test_logits_match_the_single_sequence_model(served, tiny_file):
    from lumina_b200.engine import CudaChatModel
    _, reqs, outs, steps = served
    got = {w: row for logits, who in steps for row, w in zip(logits, who)}
    m = CudaChatModel.from_lumina(tiny_file, synthetic.hf_cfg(CFG), None, theta=CFG["rope_theta"], max_seq=256, max_rows=160)
    try:
        for i, r in enumerate(reqs):
            m.kv_truncate(0)
            want = m.forward(r.prompt, 0)[0]
            for n, t in enumerate(outs[i]):
                row = got[(i, n)]
                assert np.linalg.norm(row - want) < TOL * np.linalg.norm(want), (i, n)
                seen, x = r.prompt + outs[i][:n], row.astype(np.float64).copy()
                for s in set(seen):  # the choice, from this step's own logits
                    x[s] = x[s] / r.repeat_penalty if x[s] > 0 else x[s] * r.repeat_penalty
                    x[s] -= r.frequency * seen.count(s) + r.presence
                for s, b in r.bias.items():
                    x[s] += b
                if r.allowed is not None:
                    x[~r.allowed] = -np.inf
                assert x[t] >= x.max() - 1e-5 * abs(x.max()), (i, n)
                want, _ = m.decode_step(t)
                want = np.array(want)
    finally:
        m.close()


def test_out_of_pages(tiny_file):
    import serve_batch as sb
    model = sb.BatchModel(tiny_file, CFG["num_attention_heads"], CFG["num_key_value_heads"], CFG["rope_theta"], n_pages=2)
    with pytest.raises(RuntimeError, match="out of pages"):
        model.serve([sb.Request([1] * 40)])


def test_prompts_past_the_tables_are_refused(tiny_file):
    import serve_batch as sb
    model = sb.BatchModel(tiny_file, CFG["num_attention_heads"], CFG["num_key_value_heads"], CFG["rope_theta"], max_seq=64)
    for n in (0, 65):
        with pytest.raises(ValueError, match="prompt"):
            model.serve([sb.Request([1] * 5), sb.Request([1] * n)])
    out = model.serve([sb.Request([1] * 64, max_tokens=3), sb.Request([1] * 63, max_tokens=3)])
    assert [len(o) for o in out] == [1, 2]  # the tables end there
    assert len(model.free) == 256


def test_pages_return_when_the_pool_runs_dry(tiny_file):
    import serve_batch as sb
    model = sb.BatchModel(tiny_file, CFG["num_attention_heads"], CFG["num_key_value_heads"], CFG["rope_theta"], n_pages=4)
    with pytest.raises(RuntimeError, match="out of pages"):
        model.serve([sb.Request([1] * 20), sb.Request([1] * 50)])
    assert sorted(model.free) == list(range(4))
    assert len(model.serve([sb.Request([1] * 20, max_tokens=2)])[0]) == 2


def test_steps_that_give_no_token(tiny_file):
    """A prompt of several chunks with nothing beside it."""
    import serve_batch as sb
    model = sb.BatchModel(tiny_file, CFG["num_attention_heads"], CFG["num_key_value_heads"], CFG["rope_theta"], n_pages=16)
    prompt = np.random.default_rng(5).integers(0, CFG["vocab_size"], 100).tolist()
    whole = model.serve([sb.Request(prompt, max_tokens=1)], chunk=128)
    assert model.serve([sb.Request(prompt, max_tokens=1)], chunk=30) == whole


@pytest.mark.parametrize("rows", [3, 100])
def test_a_step_with_a_fault_gives_no_tokens(tiny_file, rows):
    """A page number out of range, made on the host: the kernels report it."""
    import serve_batch as sb
    from lumina_b200 import cuda
    model = sb.BatchModel(tiny_file, CFG["num_attention_heads"], CFG["num_key_value_heads"], CFG["rope_theta"], n_pages=8)
    model.grow = lambda r, n: setattr(r, "pages", [10 ** 6] * 10)
    r = sb.Request([1] * rows)
    with pytest.raises(RuntimeError, match="fault word 64"):
        model.serve([r], chunk=64)
    assert r.out == [] and cuda.fault_status(0) == 0


def test_requests_of_equal_fields(tiny_file):
    """The same prompt twice, under different masks: each ends by itself."""
    import serve_batch as sb
    model = sb.BatchModel(tiny_file, CFG["num_attention_heads"], CFG["num_key_value_heads"], CFG["rope_theta"], n_pages=16)
    masks = np.zeros((2, CFG["vocab_size"]), bool)
    masks[0, 5] = masks[1, 9] = True
    out = model.serve([sb.Request([1, 2, 3], max_tokens=2, allowed=m) for m in masks])
    assert out == [[5, 5], [9, 9]]
    assert not (sb.Request([1], allowed=masks[0]) == sb.Request([1], allowed=masks[1]))
    one, two = sb.Request([1]), sb.Request([1])
    live = [one, two]
    live.remove(two)
    assert live[0] is one
