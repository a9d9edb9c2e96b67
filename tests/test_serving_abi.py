"""The serving entry points without a device: null contexts and handles are
refused, not dereferenced."""

import ctypes as C

from llm_mojo_b200 import _lib, build


def test_null_arguments_are_refused():
    build.build()
    L = _lib.lib()
    h = C.c_void_p()
    assert L.llmq_paged_create(None, _lib.KV_QUANT8, 1, 1, 16, 1, 64, C.byref(h)) == _lib.ERR_INVALID
    assert L.llmq_paged_free(None) == _lib.ERR_INVALID
    assert L.llmq_paged_buffers(None, None, None, None, None) == _lib.ERR_INVALID
    assert L.llmq_paged_store(None, None, 0, None, 0, None, 0, None, None, 1, None, 1, 1, 1) == _lib.ERR_INVALID
    assert L.llmq_paged_attend(None, None, 0, None, 0, None, 0, 1, 1, None, 1, 1, None, 1, 1.0, None, None,
                               0) == _lib.ERR_INVALID
    assert L.llmq_paged_evict(None, None, 0, 1, 1, None, 1, 1, None, 1, None, 1, 1, 0, 0, None, 1, 1, None, None, 1,
                              None) == _lib.ERR_INVALID
    assert L.llmq_process_logits(None, None, 0, None, 0, 1, 1, None, None) == _lib.ERR_INVALID


def test_rules_struct_matches_the_header():
    """The ctypes struct has the header's fields in the header's order."""
    import os
    import re

    from llm_mojo_b200.serving import _Rules

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = open(os.path.join(root, "include", "llmq.h")).read()
    body = re.search(r"typedef struct llmq_logit_rules \{(.*?)\}", text, flags=re.S).group(1)
    names = []
    for decl in body.split(";"):
        decl = decl.strip()
        if decl:
            names += [x.strip(" *") for x in re.sub(r"^(const )?(float|int|long long|uint32_t) ", "", decl).split(",")]
    assert names == [f[0] for f in _Rules._fields_]


def test_pack_mask():
    import torch

    from llm_mojo_b200.paged_generate import pack_mask

    g = torch.Generator().manual_seed(1)
    for V in (1, 31, 32, 33, 100):
        ok = torch.rand(3, V, generator=g) < 0.5
        ok[0, V - 1] = True
        words = pack_mask(ok)
        assert words.shape == (3, (V + 31) // 32) and words.dtype == torch.int32
        for r in range(3):
            assert [bool(int(words[r, t // 32]) >> (t % 32) & 1) for t in range(V)] == ok[r].tolist()


def test_page_pool():
    import pytest

    from llm_mojo_b200.paged_generate import PagePool

    p = PagePool(4)
    a, b = p.take(3), p.take(1)
    assert sorted(a + b) == [0, 1, 2, 3]
    with pytest.raises(RuntimeError):
        p.take(1)
    p.give(a)
    assert sorted(p.take(3)) == sorted(a)
