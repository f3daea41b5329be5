"""The models and the block loop over paged caches (stack.py, spec_decode.py with ``page_size``): logits against the
ragged path, output ids and acceptance lengths against the reference's own (tests/golden/spec_loop_*.npz)."""
import numpy as np
import pytest
import torch

from tests.fixtures import LOOP_CASES, load_loop

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available() or torch.cuda.get_device_capability(0)[0] != 10:
        pytest.fail("GPU tests need an sm_100 device")


def _runner(draft, target, B):
    from domino_b200 import DraftCorrectionGraphRunner

    cfg = draft.cfg
    P = cfg.pure_draft_prefix_len
    return DraftCorrectionGraphRunner(draft, target, B, 15 - P, cfg.hidden_size, cfg.gru_hidden_dim, cfg.vocab_size, 1 + P,
                                      torch.device("cuda", 0))


@pytest.mark.parametrize("page_size", [16, 64])
@pytest.mark.parametrize("case", LOOP_CASES)
def test_paged_loop_matches_reference(case, page_size):
    from domino_b200.spec_decode import spec_generate

    c = load_loop(case, device="cuda")
    draft, target = c["draft"], c["target"]
    r = _runner(draft, target, 1)
    res = spec_generate(draft, target, r, c["prompts"][:1], c["max_new_tokens"], page_size=page_size)
    assert np.array_equal(res.output_ids[0].cpu().numpy(), c["outputs"][0])
    assert res.acceptance_lengths[0] == c["accepts"][0]
    r = _runner(draft, target, 3)
    res = spec_generate(draft, target, r, c["prompts"], c["max_new_tokens"], page_size=page_size)
    assert r.status() == 0
    for i in range(3):
        assert np.array_equal(res.output_ids[i].cpu().numpy(), c["outputs"][i]), i
        assert res.acceptance_lengths[i] == c["accepts"][i], i


def test_shared_prefix_loop_matches_separate_prompts():
    """Prompts that begin alike, prefilled once and forked: the same ids and acceptance as each prompt's own prefill."""
    from domino_b200.spec_decode import spec_generate

    c = load_loop("spec_loop_varied", device="cuda")
    draft, target = c["draft"], c["target"]
    head = torch.cat([c["prompts"][0], c["prompts"][1]])[:21].cpu()
    prompts = [torch.cat([head, t.cpu()[: 3 + 4 * i]]) for i, t in enumerate(c["prompts"])]
    r = _runner(draft, target, 3)
    a = spec_generate(draft, target, r, prompts, 40, page_size=16, share_prefix=True)
    b = spec_generate(draft, target, r, prompts, 40)
    for i in range(3):
        assert torch.equal(a.output_ids[i], b.output_ids[i])
    assert a.acceptance_lengths == b.acceptance_lengths
    with pytest.raises(ValueError):
        spec_generate(draft, target, r, prompts, 40, share_prefix=True)


@pytest.mark.parametrize("kw", [dict(), dict(sliding_window=9, sink_tokens=2),
                                dict(sliding_window=20, window_layers=[False, True]),
                                dict(rope_scaling={"rope_type": "yarn", "factor": 4.0,
                                                   "original_max_position_embeddings": 32})])
def test_paged_target_matches_ragged_target(kw):
    """fp32 logits of prompts of different length, then a block: both paths compute in fp32 and differ by roundings of
    2^-24 (GEMMs and sums in another order), 1e-4 of logits of order one is far above and far below any wrong key."""
    from domino_b200.stack import StackConfig, TargetLM

    torch.manual_seed(1)
    cfg = StackConfig(vocab_size=211, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=6,
                      num_key_value_heads=2, head_dim=24, rope_theta=1e4, **kw)
    prev = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    try:
        t = TargetLM(cfg).cuda().eval()
        a, b = t.new_cache(2, 120), t.new_cache(2, 120, page_size=16)
        ids = torch.randint(0, 211, (2, 50), device="cuda")
        valid = torch.arange(50, device="cuda")[None] < torch.tensor([[50], [33]], device="cuda")
        for step_ids, step_valid in ((ids, valid), (ids[:, :16], torch.ones(2, 16, dtype=torch.bool, device="cuda")),
                                     (ids[:, :1], torch.ones(2, 1, dtype=torch.bool, device="cuda"))):
            la, _ = t(step_ids, a, step_valid)
            lb, _ = t(step_ids, b, step_valid)
            assert (la - lb)[step_valid].abs().max() <= 1e-4 * la.abs().max()
        assert b.status() == 0 and a.length.tolist() == b.length.tolist()
    finally:
        torch.backends.cuda.matmul.allow_tf32 = prev


def test_bf16_target_paged_close_to_ragged():
    """bf16: the paths round at different places (2^-8 each), so logits agree to a few of those."""
    from domino_b200.stack import StackConfig, TargetLM

    torch.manual_seed(2)
    cfg = StackConfig(vocab_size=211, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=8,
                      num_key_value_heads=2, head_dim=128)
    t = TargetLM(cfg).cuda().to(torch.bfloat16).eval()
    a, b = t.new_cache(2, 400), t.new_cache(2, 400, page_size=64)
    ids = torch.randint(0, 211, (2, 300), device="cuda")
    ok = torch.ones_like(ids, dtype=torch.bool)
    la, _ = t(ids, a, ok)
    lb, _ = t(ids, b, ok)
    # about 10 roundings of 2^-8 per layer on the residual path, two layers
    assert (la.float() - lb.float()).abs().max() <= 20 * 2.0 ** -8 * la.float().abs().max()
