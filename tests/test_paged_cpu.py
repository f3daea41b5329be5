"""Refusals of the paged cache and its operators, and the rotary frequencies: no GPU needed."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from domino_b200.build import build
    build()
    from domino_b200 import _lib
    return _lib.load()


def shape(**kw):
    from domino_b200 import _lib
    base = dict(layers=1, batch=2, kv_heads=2, pages=4, page_size=64, head_dim=64, row_pages=2, dtype=_lib.DD_BF16)
    base.update(kw)
    return _lib.DDPagedCache(**base)


def full(**kw):
    """A cache struct whose pointers are aligned numbers: nothing is read before a refusal."""
    c = shape(**kw)
    c.data = c.scratch = 1 << 20
    c.table = c.length = c.refs = c.status = 1 << 20
    return c


@pytest.mark.parametrize("bad", [dict(layers=0), dict(batch=0), dict(batch=1025), dict(kv_heads=0), dict(pages=0),
                                 dict(row_pages=0), dict(page_size=48), dict(page_size=8), dict(page_size=256),
                                 dict(head_dim=0), dict(head_dim=12), dict(head_dim=264), dict(dtype=7),
                                 dict(pages=1 << 30, kv_heads=4), dict(batch=1024, row_pages=1 << 22), dict(row_pages=(1 << 24) + 1)])
def test_cache_shapes_refused(lib, bad):
    from domino_b200 import PagedKVCache, _lib
    n = ctypes.c_uint64()
    assert lib.dd_cache_scratch(ctypes.byref(shape(**bad)), ctypes.byref(n)) == _lib.DD_EINVAL
    assert b"paged cache" in lib.dd_last_error(None)
    if "dtype" not in bad:
        args = dict(layers=1, batch=2, kv_heads=2, pages=4, head_dim=64, dtype=torch.bfloat16, device="cuda", row_pages=2)
        args.update(bad)
        with pytest.raises(ValueError):
            PagedKVCache(**args)


def test_cache_refuses_types_and_devices(lib):
    from domino_b200 import PagedKVCache
    with pytest.raises(NotImplementedError):
        PagedKVCache(1, 1, 1, 1, 64, torch.float64, "cuda")
    with pytest.raises(RuntimeError):
        PagedKVCache(1, 1, 1, 1, 64, torch.bfloat16, "cpu")


def test_calls_refuse_null_and_misaligned_pointers(lib):
    from domino_b200 import _lib
    x = ctypes.c_void_p(1 << 20)
    for call in (lib.dd_pages_reserve, lib.dd_pages_crop, lib.dd_pages_fork):
        assert call(None, x, None) == _lib.DD_EINVAL
        assert call(ctypes.byref(shape()), x, None) == _lib.DD_EINVAL
        assert call(ctypes.byref(full()), None, None) == _lib.DD_EINVAL
    assert lib.dd_pages_compact(ctypes.byref(shape()), None) == _lib.DD_EINVAL
    c = full()
    c.data = (1 << 20) + 8
    assert lib.dd_pages_crop(ctypes.byref(c), x, None) == _lib.DD_EINVAL
    assert b"aligned" in lib.dd_last_error(None)


@pytest.mark.parametrize("bad", [dict(layer=1), dict(layer=-1), dict(tokens=0), dict(heads=0), dict(heads=3),
                                 dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(window=-1), dict(sinks=1), dict(window=4, causal=0), dict(window=4, sinks=-1),
                                 dict(q=None), dict(out=None), dict(start=None), dict(out=(1 << 20) + 4)])
def test_attend_arguments_refused(lib, bad):
    from domino_b200 import _lib
    args = dict(q=1 << 20, out=1 << 20, start=1 << 20, scale=1.0, layer=0, tokens=4, heads=4, causal=1, window=0, sinks=0)
    args.update(bad)
    a = _lib.DDCacheAttendArgs(**args)
    assert lib.dd_cache_attend(ctypes.byref(full()), ctypes.byref(a), None) == _lib.DD_EINVAL


@pytest.mark.parametrize("bad", [dict(layer=1), dict(tokens=0), dict(rotary=3), dict(rotary=66), dict(rotary=-2),
                                 dict(inv_freq=None), dict(k=None), dict(v=None), dict(start=None), dict(q_out=None),
                                 dict(q_out=(1 << 20) + 2), dict(heads=0)])
def test_write_arguments_refused(lib, bad):
    from domino_b200 import _lib
    args = dict(q=1 << 20, k=1 << 20, v=1 << 20, q_out=1 << 20, start=1 << 20, inv_freq=1 << 20, eps=1e-6, factor=1.0,
                layer=0, tokens=4, heads=4, rotary=64)
    args.update(bad)
    a = _lib.DDCacheWriteArgs(**args)
    assert lib.dd_cache_write(ctypes.byref(full()), ctypes.byref(a), None) == _lib.DD_EINVAL


def test_rope_refusals():
    from domino_b200 import Rope
    for kw in (dict(rotary_dim=3), dict(rotary_dim=66), dict(rotary_dim=4, inv_freq=torch.ones(3)),
               dict(inv_freq=torch.ones(33)), dict(inv_freq=torch.ones(2, 2)),
               dict(inv_freq=torch.ones(2), scaling={"rope_type": "linear", "factor": 2.0})):
        with pytest.raises(ValueError):
            Rope(64, **kw)
    with pytest.raises(NotImplementedError):
        Rope(64, scaling={"rope_type": "dynamic", "factor": 2.0})


@pytest.mark.parametrize("scaling", [
    {"rope_type": "default"},
    {"rope_type": "linear", "factor": 4.0},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
    {"rope_type": "yarn", "factor": 2.0, "original_max_position_embeddings": 4096, "beta_fast": 16, "beta_slow": 2,
     "attention_factor": 1.5},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 8192}])
def test_rope_frequencies_match_transformers(scaling):
    """The scaled frequencies against transformers' own (fp32 both: a few roundings of 2^-24)."""
    from transformers import Qwen3Config
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS

    from domino_b200 import Rope

    r = Rope(128, theta=1e6, scaling=scaling)
    cfg = Qwen3Config(hidden_size=1024, num_attention_heads=8, head_dim=128, max_position_embeddings=131072)
    cfg.rope_parameters = {"rope_theta": 1e6, **scaling}
    if scaling["rope_type"] == "default":
        inv, factor = 1e6 ** -(torch.arange(0, 128, 2, dtype=torch.float64) / 128), 1.0
    else:
        inv, factor = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu")
    assert torch.allclose(r.inv_freq.double(), inv.double(), rtol=8 * 2.0 ** -24, atol=0)
    assert abs(r.factor - factor) < 1e-6


def _tiny(**kw):
    from transformers import Qwen3Config
    return Qwen3Config(vocab_size=97, hidden_size=32, intermediate_size=48, num_hidden_layers=3, num_attention_heads=4,
                       num_key_value_heads=2, head_dim=16, max_position_embeddings=64, **kw)


@pytest.mark.parametrize("kw", [
    dict(rope_parameters={"rope_theta": 1e4, "rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 16}),
    dict(rope_parameters={"rope_theta": 1e4, "rope_type": "linear", "factor": 2.0}),
    dict(use_sliding_window=True, sliding_window=5, max_window_layers=0),
    dict(use_sliding_window=True, sliding_window=7, layer_types=["full_attention", "sliding_attention", "full_attention"])])
def test_long_context_config_matches_transformers(kw):
    """TargetLM with a config's scaled frequencies or sliding-window layers against transformers' Qwen3 (fp32 both: a
    few operations of 2^-24 on values of order one)."""
    from transformers import Qwen3ForCausalLM

    from domino_b200.stack import StackConfig, TargetLM

    torch.manual_seed(0)
    cfg = _tiny(**kw)
    cfg._attn_implementation = "eager"
    hf = Qwen3ForCausalLM(cfg).eval()
    c = StackConfig.from_hf(cfg, long_context=True)
    assert (c.rope_scaling is not None) == ("rope_parameters" in kw) and (c.sliding_window > 0) == ("sliding_window" in kw)
    plain = StackConfig.from_hf(cfg)
    assert plain.rope_scaling is None and plain.sliding_window == 0
    t = TargetLM(c).eval()
    t.load_state_dict(hf.state_dict())
    ids = torch.randint(0, 97, (1, 40))
    with torch.no_grad():
        ref = hf(ids).logits
    cache = t.new_cache(1, 64)
    got = torch.cat([t(part, cache, torch.ones_like(part, dtype=torch.bool))[0] for part in ids.split([25, 1, 14], dim=1)], 1)
    assert torch.allclose(got, ref, atol=1e-5, rtol=1e-5)


def test_paged_caches_need_a_gpu_and_a_page_size():
    from domino_b200.spec_decode import common_prefix
    from domino_b200.stack import StackConfig, TargetLM

    t = TargetLM(StackConfig.from_hf(_tiny()))
    with pytest.raises(RuntimeError):
        t.new_cache(1, 64, page_size=16)
    p = torch.arange(10)
    assert common_prefix([p, p]) == 9
    assert common_prefix([p]) == 9
    assert common_prefix([p, torch.tensor([0, 1, 2, 9, 9])]) == 3
    assert common_prefix([p, torch.tensor([1])]) == 0
