"""The paged cache without a GPU: calls refused for their size, and what the block loop does with its caches' errors."""
import ctypes

import numpy as np
import pytest
import torch

from tests.fixtures import LOOP_CASES, load_loop
from tests.test_paged_cpu import full, lib  # noqa: F401 (a fixture)
from tests.test_spec_loop_cpu import OracleRunner


@pytest.mark.parametrize("heads,dim,ok", [(1 << 23, 256, False), (1 << 24, 256, False), ((1 << 28) - 1, 8, True),
                                          (1 << 28, 8, False), ((1 << 23) - 1, 256, True)])
def test_write_refuses_tokens_of_2_31_query_values(lib, heads, dim, ok):  # noqa: F811
    """The kernel counts a token's query values in 32 bits; without a GPU an accepted call fails at the device instead."""
    from domino_b200 import _lib

    a = _lib.DDCacheWriteArgs(q=1 << 20, k=1 << 20, v=1 << 20, q_out=1 << 20, start=1 << 20, inv_freq=1 << 20, eps=1e-6,
                              factor=1.0, layer=0, tokens=1, heads=heads, rotary=8)
    c = full(head_dim=dim)
    c.device = 63  # no such device: nothing is launched on a machine with a GPU either
    rc = lib.dd_cache_write(ctypes.byref(c), ctypes.byref(a), None)
    assert rc < 0 and (rc == _lib.DD_EINVAL) != ok
    assert (b"chunk too large" in lib.dd_last_error(None)) != ok


@pytest.mark.parametrize("bits,who,name", [((8, 0), "target", "DD_STATUS_NO_PAGE"), ((0, 33), "drafter", "DD_STATUS_TIMEOUT"),
                                           ((0, 33), "drafter", "DD_STATUS_SHARED_PAGE"), ((0, 0), None, None)])
def test_the_loop_raises_what_its_paged_caches_report(bits, who, name):
    """Status bits of the caches that the loop makes come out as an error, not as tokens."""
    from domino_b200 import DominoDraftError
    from domino_b200.spec_decode import spec_generate
    from domino_b200.stack import RaggedKVCache

    class Cache(RaggedKVCache):  # the padded cache with a paged one's two calls
        reads = 0

        def crop(self, length):
            self.length.copy_(torch.minimum(self.length, length))

        def status(self):
            self.reads += 1
            return self.bits

    c = load_loop(LOOP_CASES[0])
    draft, target = c["draft"], c["target"]
    made = []
    for model, b in ((target, bits[0]), (draft, bits[1])):
        def new_cache(batch, capacity, page_size=0, model=model, b=b):
            assert page_size == 16
            cfg = model.cfg
            cache = Cache(cfg.num_hidden_layers, batch, cfg.num_key_value_heads, capacity, cfg.head_dim,
                          next(model.parameters()).dtype, "cpu")
            cache.bits = b
            made.append(cache)
            return cache

        model.new_cache = new_cache
    runner = OracleRunner(draft, target, 1, draft.cfg.pure_draft_prefix_len)
    go = lambda: spec_generate(draft, target, runner, c["prompts"][:1], c["max_new_tokens"], page_size=16)  # noqa: E731
    if who:
        with pytest.raises(DominoDraftError, match=f"{who}.*{name}"):
            go()
    else:
        assert np.array_equal(go().output_ids[0].numpy(), c["outputs"][0])
        assert [x.reads for x in made] == [1, 1]
