"""Stored prefixes, forks and samples over 4-bit pages, where they meet other formats, full caches and many settings."""
import pytest
import torch

from test_kv4_engine import _load, _prompt


@pytest.mark.parametrize("order", [("bf16", "affine4"), ("affine4", "bf16")])
def test_one_store_holds_a_prompt_in_both_formats(tmp_path, order):
    """The formats share a directory of stored prefixes: each stores a prompt of its own there, and finds it again."""
    ids, want = _prompt(70), {}
    for kv_format in order + order:
        m = _load("cpu", kv_format=kv_format, prefix_cache=True, runtime_dir=str(tmp_path))
        first = m.prefill(ids)
        store, again = m.prefix_store(), kv_format in want
        assert (store.stored, store.hits) == ((0, 1) if again else (1, 0))
        got = [first] + [m.decode() for _ in range(3)]
        assert got == want.setdefault(kv_format, got)
