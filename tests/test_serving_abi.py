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
