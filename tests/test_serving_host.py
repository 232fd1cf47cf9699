"""Host side of the batched serving calls: layout sizes, the ctypes structs
against the header, and what is refused before any GPU work."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

import serving_ref as ref
from lumina_b200 import cuda, serving
from lumina_b200.cuda import LuminaError

HEADER = open(os.path.join(os.path.dirname(__file__), "..", "include", "lumina_cuda.h")).read()
C_TYPES = {"int": ctypes.c_int, "float": ctypes.c_float, "size_t": ctypes.c_size_t}


@pytest.mark.parametrize("name,cls", [("lumina_kvq_pool", serving._Pool), ("lumina_kvq_batch", serving._Batch),
                                      ("lumina_kvq_attend_args", serving._Attend), ("lumina_logits_args", serving._Logits)])
def test_structs_match_the_header(name, cls):
    body = re.search(r"typedef struct \{([^{}]*)\} %s;" % name, HEADER).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    want = []
    for decl in body.split(";"):
        decl = " ".join(decl.split())
        if not decl:
            continue
        first, *rest = decl.split(",")
        base, field = re.match(r"(?:const )?(\w+) ?(\*?\w+)$", re.sub(r" ?\* ?", " *", first)).groups()
        for f in [field] + [r.strip() for r in rest]:
            want.append((f.lstrip("* "), ctypes.c_void_p if f.startswith("*") else C_TYPES[base]))
    assert [(n, t) for n, t in cls._fields_] == want


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
def test_block_bytes(bits, hd, page):
    assert serving.KVPool.block_bytes(bits, hd, page) == ref.block_bytes(bits, hd, page) == page * (2 * hd * bits // 8 + 8)


@pytest.mark.parametrize("bits,hd,page", [(2, 64, 16), (16, 64, 16), (8, 0, 16), (8, 12, 16), (8, 64, 0), (4, -8, 16)])
def test_block_bytes_refusals(bits, hd, page):
    with pytest.raises(LuminaError):
        serving.KVPool.block_bytes(bits, hd, page)


def test_null_arguments_are_errors():
    lib = cuda.bound_lib()
    assert lib.lumina_kvq_block_bytes(8, 64, 16, None) != 0
    assert lib.lumina_kvq_workspace_bytes(0, None) != 0
    assert lib.lumina_kvq_append(None, None, None, 0, None, 0, None, 0, 0, 1, None, None, 0.0, None, None, 1, None, 0, None) != 0
    assert lib.lumina_kvq_read(None, None, None, None, 0, 0, None) != 0
    assert lib.lumina_kvq_attend(None, None, None, None) != 0
    assert lib.lumina_logits_adjust(None, None) != 0
    assert "null" in cuda.last_error(lib)


def test_cpu_tensors_are_refused():
    i32 = torch.int32
    with pytest.raises(LuminaError, match="CUDA tensor"):
        serving.KVPool(torch.zeros(2, 1, 16 * 136, dtype=torch.uint8), 8, 64, 16)
    with pytest.raises(LuminaError, match="CUDA tensors"):
        serving.SeqBatch(torch.zeros(2, dtype=i32), torch.zeros(1, dtype=i32), torch.zeros(1, 1, dtype=i32), 1, 1)
    with pytest.raises(LuminaError, match="on the GPU"):
        serving.adjust_logits(torch.zeros(1, 8))


def test_the_plain_attention_by_differences():
    """The oracle's masks: what a key weighs shows in the output's change
    when its value moves."""
    rng = np.random.default_rng(0)
    n, ln, hd, window, pre = 3, 9, 4, 2, 3
    q, k, v = rng.standard_normal((n, 2, hd)), rng.standard_normal((ln, 1, hd)), rng.standard_normal((ln, 1, hd))
    base = ref.attend(q, k, v, ln, 0.5, window=window, prefix=pre)
    for j in range(ln):
        w = v.copy()
        w[j] += 1.0
        moved = np.abs(ref.attend(q, k, w, ln, 0.5, window=window, prefix=pre) - base).max(axis=(1, 2)) > 1e-9
        assert moved.tolist() == [j < pre or (p - window < j <= p) for p in range(ln - n, ln)]


def test_vocabularies_past_int_tokens_are_refused():
    """Before any GPU work: a token plus a chunk of tokens would pass 31 bits."""
    lib = cuda.bound_lib()
    a = serving._Logits(16, 16, 2 ** 31 - 1, 2 ** 31 - 1, 1, 2 ** 30 + 1)
    assert lib.lumina_logits_adjust(ctypes.byref(a), None) == 1
    assert str(2 ** 30 + 1) in cuda.last_error(lib)
