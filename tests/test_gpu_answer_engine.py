"""MkEngine's answers from its own operators: score() against generate() and the logits, and the 4-bit head."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32 = torch.float32


@pytest.fixture(scope="module")
def engines():
    from minicpm5_mk.config import preset
    from minicpm5_mk.engine import MkEngine
    from minicpm5_mk.synth import random_hf_state_dict

    cfg = preset("tiny")
    sd = random_hf_state_dict(cfg)
    kw = dict(quant="auto", state_dict=sd, max_model_len=1024, device="cuda:0", log=lambda *a: None, precompile="")
    pair = MkEngine(cfg, **kw), MkEngine(cfg, lm_head_quant="w4", **kw)
    yield pair, sd
    for e in pair:
        e.close()


def _prompts(bs=3, seq=256):
    from minicpm5_mk.synth import random_token_ids

    return [r.tolist() for r in random_token_ids(bs, seq)]


def test_score_matches_generate(engines):
    """The same log probabilities and tokens as generate's, which torch makes in f32: 2^-24 a rounding, 64 of them."""
    from minicpm5_mk.engine import SamplingParams

    (eng, _), _ = engines
    ps = _prompts()
    outs = eng.generate([{"prompt_token_ids": p} for p in ps], SamplingParams(max_tokens=1, temperature=0.0, logprobs=20))
    r = eng.score([{"prompt_token_ids": p} for p in ps], candidates=[[o.outputs[0].token_ids[0], 7] for o in outs], top=20)
    for b, o in enumerate(outs):
        tok, lps = o.outputs[0].token_ids[0], o.outputs[0].logprobs[0]
        assert int(r.top_ids[b, 0]) == tok and int(r.ranks[b, 0]) == 1
        assert set(r.top_ids[b].tolist()) == set(lps)
        for i, v in zip(r.top_ids[b].tolist(), r.top_logprobs[b].tolist()):
            assert abs(v - lps[i]) <= 64 * 2.0 ** -24 * (1 + abs(v))
    lg = eng.logits(torch.tensor(ps, dtype=torch.int32)).double()
    want = torch.log_softmax(lg, -1)
    assert float((r.token_logprobs[:, 1].double() - want[:, 7]).abs().max()) <= 400 * 2.0 ** -24 * (1 + float(want.abs().max()))
    assert torch.equal(r.ranks[:, 1].long(), 1 + (lg > lg[:, 7:8]).sum(-1) + (lg[:, :7] == lg[:, 7:8]).sum(-1))


def test_score_forms(engines):
    from minicpm5_mk.engine import NotEligible

    (eng, _), _ = engines
    ps = _prompts(2)
    a, b = eng.score(ps, candidates=[3, 9, 1]), eng.score(ps, candidates=[[3, 9, 1], [3, 9, 1]])
    assert torch.equal(a.token_logprobs, b.token_logprobs) and a.top_ids is None and a.token_logprobs.shape == (2, 3)
    c = eng.score(ps, top=4)
    assert c.token_logprobs is None and c.top_ids.shape == (2, 4) and torch.equal(c.entropy, a.entropy)
    with pytest.raises(NotEligible, match="ragged"):
        eng.score([ps[0], ps[1][:128]])
    with pytest.raises(ValueError, match="token ids"):
        eng.score(ps, candidates=[eng.cfg.vocab])


def test_w4_head(engines):
    """The engine with a 4-bit head: the logits of its hidden rows and the weights it stands for."""
    from minicpm5_mk import ops
    from minicpm5_mk.engine import SamplingParams

    (plain, eng), sd = engines
    ps = _prompts()
    ids = torch.tensor(ps, dtype=torch.int32)
    lg = eng.logits(ids).clone()
    hidden = eng.model.forward(ids.cuda().reshape(-1), 3, 256)[:3]
    assert torch.equal(hidden, plain.model.forward(ids.cuda().reshape(-1), 3, 256)[:3])
    head = ops.dequantize_w4(eng.lm_head_w4, dtype=F32)
    assert torch.equal(head, ops.dequantize_w4(ops.quantize_w4(sd["lm_head.weight"].to("cuda", torch.bfloat16), 64), dtype=F32))
    want = torch.mm(hidden.double(), head.double().T.contiguous())
    assert float((lg.double() - want).norm()) <= 4e-6 * float(want.norm())
    # the head's own rounding moves the logits by a few percent of their spread, no more: codes are off by half a step of
    # a seventh of a group's largest weight, 64 values of which reach about 2.4 sigma
    base = plain.logits(ids).double()
    assert float((lg.double() - base).norm()) <= 0.2 * float((base - base.mean()).norm())
    r = eng.score(ps, candidates=[1, 2], top=3)
    lp = torch.log_softmax(want, -1)
    assert float((r.token_logprobs.double() - lp[:, [1, 2]]).abs().max()) <= 1e-4
    outs = eng.generate([{"prompt_token_ids": p} for p in ps], SamplingParams(max_tokens=1, temperature=0.0))
    assert [o.outputs[0].token_ids[0] for o in outs] == lg.argmax(-1).tolist() == r.top_ids[:, 0].tolist()


def test_w4_head_precompile(engines):
    from minicpm5_mk.config import preset
    from minicpm5_mk.engine import MkEngine

    _, sd = engines
    eng = MkEngine(preset("tiny"), quant="auto", state_dict=sd, max_model_len=1024, device="cuda:0", log=lambda *a: None,
                   precompile="3x256", lm_head_quant="w4")
    assert eng.model.graph_count() == 1
    ps = _prompts()
    a = eng.score(ps, top=2)
    assert eng.model.graph_count() == 1
    b = eng.score(ps, top=2)
    assert torch.equal(a.top_logprobs, b.top_logprobs)
    eng.close()
