"""The attention operators' entry points without a GPU: every refusal is made before anything is queued."""
import ctypes as C
import re
import os

import pytest
import torch

from conftest import ROOT
from vesper_db_b200 import _native as N
from vesper_db_b200 import attention as A
from vesper_db_b200.index import VesperError

P = 1 << 20  # a 16-byte aligned address that nothing reads: each call below is refused


def refused(fn, params):
    lib = N.load()
    status = getattr(lib, fn)(params, None)
    assert status == N.VESPER_ERROR_INVALID_PARAM
    return lib.vesper_get_last_error().decode()


FIELDS = {
    "page_tables": (A._TABLES, [P, P, 4, P, 9, P, 5, 5, 16, 8, 0, P, P, P, P, P]),
    "norm_rotate": (A._ROTATE, [0, 8, 8, 2, 128, 128, 0, 1e-6, P, 1024, 128, P, 256, 128, P, 256, 128, P, P, 99, P, P, P, P,
                                4096, 256, 128, P, 4096, 256, 128, 7, 16, P, P]),
    "prompt_attention": (A._PROMPT, [0, 2, 8, 8, 8, 2, 128, 1, 0.1, P, 1024, 128, P, 256, 128, P, 256, 128, P, P, P, P, 0, 0]),
    "shared_prefix_attention": (A._SHARED, [0, 4, 8, 2, 128, 0.1, P, 1024, 128, P, 4096, 256, 128, P, 4096, 256, 128, 7, 16, P,
                                            20, P, 5, 5, P, P, P, 0, 0]),
}


def test_packed_structs_match_the_header():
    """One 8-byte field for each member that the header declares, in its order."""
    text = open(os.path.join(ROOT, "include", "vesper_b200.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, (packed, fields) in FIELDS.items():
        body = re.search(r"typedef struct vesper_%s_params_s \{(.*?)\}" % name, text, re.S).group(1)
        kinds = []
        for line in body.split(";"):
            if line.strip():
                first, *more = line.split(",")
                kinds += ["d" if first.split()[0] == "double" else "q"] * (1 + len(more))
                assert "*" in line or first.split()[0] in ("size_t", "int64_t", "double"), line
        assert packed.size == 8 * len(kinds) == 8 * (1 + len(fields)), name
        assert ["d" if isinstance(f, float) else "q" for f in fields] == kinds[1:], name


@pytest.mark.parametrize("name,at,value,says", [
    ("page_tables", 8, 15, "page_size"), ("page_tables", 8, 512, "page_size"), ("page_tables", 8, 48, "page_size"),
    ("page_tables", 2, 16385, "requests"), ("page_tables", 0, 0, "d_cached"), ("page_tables", 3, 0, "d_free"),
    ("page_tables", 5, 0, "d_table"), ("page_tables", 7, 4, "table_stride"), ("page_tables", 9, 1 << 31, "sizes"),
    ("page_tables", 10, -1, "base"), ("page_tables", 12, 0, "d_starts"), ("page_tables", 14, 0, "d_slots"),
    ("norm_rotate", 0, 2, "dtype"), ("norm_rotate", 3, 3, "multiple of kv_heads"), ("norm_rotate", 4, 260, "head_dim"),
    ("norm_rotate", 4, 264, "head_dim"), ("norm_rotate", 5, 24, "turned"), ("norm_rotate", 5, 144, "turned"),
    ("norm_rotate", 7, -1.0, "eps"), ("norm_rotate", 7, float("nan"), "eps"), ("norm_rotate", 8, P + 8, "aligned"),
    ("norm_rotate", 9, 1020, "strides"), ("norm_rotate", 11, 0, "d_k"), ("norm_rotate", 14, 0, "d_v"),
    ("norm_rotate", 17, 0, "positions"), ("norm_rotate", 18, 0, "turns"), ("norm_rotate", 20, P + 2, "weights"),
    ("norm_rotate", 23, 0, "k_cache"), ("norm_rotate", 28, 132, "strides"), ("norm_rotate", 32, 24, "page_size"),
    ("norm_rotate", 33, 0, "out_q"), ("norm_rotate", 1, 1 << 31, "sizes"),
    ("prompt_attention", 0, 7, "dtype"), ("prompt_attention", 4, 0, "heads"), ("prompt_attention", 5, 0, "heads"),
    ("prompt_attention", 6, 136, "head_dim"), ("prompt_attention", 6, 20, "head_dim"), ("prompt_attention", 8, 0.0, "scale"),
    ("prompt_attention", 8, float("inf"), "scale"), ("prompt_attention", 8, -1.0, "scale"), ("prompt_attention", 9, 0, "d_q"),
    ("prompt_attention", 10, 1028, "strides"), ("prompt_attention", 10, -1024, "strides"), ("prompt_attention", 12, P + 4, "aligned"),
    ("prompt_attention", 18, 0, "starts"), ("prompt_attention", 20, 0, "d_out"), ("prompt_attention", 2, 1 << 31, "tokens"),
    ("prompt_attention", 4, 258, "128"),
    ("shared_prefix_attention", 0, -1, "dtype"), ("shared_prefix_attention", 5, float("nan"), "scale"),
    ("shared_prefix_attention", 4, 4, "head_dim"), ("shared_prefix_attention", 6, 0, "d_q"),
    ("shared_prefix_attention", 9, P + 2, "aligned"), ("shared_prefix_attention", 14, 4097, "strides"),
    ("shared_prefix_attention", 17, 0, "no pages"), ("shared_prefix_attention", 18, 8, "page_size"),
    ("shared_prefix_attention", 19, 0, "prefix_pages"), ("shared_prefix_attention", 20, 1 << 31, "prefix_len"),
    ("shared_prefix_attention", 21, 0, "d_table"), ("shared_prefix_attention", 23, 3, "table_stride"),
    ("shared_prefix_attention", 24, 0, "lengths"), ("shared_prefix_attention", 25, P + 8, "d_out"),
    ("shared_prefix_attention", 22, 1 << 28, "table_width"),
])
def test_refusals(name, at, value, says):
    packed, fields = FIELDS[name]
    fields = list(fields)
    fields[at] = value
    msg = refused(f"vesper_{name}_device", packed.pack(packed.size, *fields))
    assert says in msg, msg


@pytest.mark.parametrize("name", list(FIELDS))
def test_struct_size_and_null(name):
    packed, fields = FIELDS[name]
    assert "struct_size" in refused(f"vesper_{name}_device", packed.pack(packed.size - 8, *fields))
    assert "NULL" in refused(f"vesper_{name}_device", None)


def test_different_lengths_need_their_starts():
    packed, fields = FIELDS["prompt_attention"]
    fields = list(fields)
    fields[3], fields[19] = 9, 0
    assert "d_starts_k" in refused("vesper_prompt_attention_device", packed.pack(packed.size, *fields))


def test_python_refuses_host_tensors():
    x, i = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(5, dtype=torch.int32)
    c = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: A.page_tables(i, i, i, torch.zeros(5, 2, dtype=torch.int32), 16, 5),
                 lambda: A.norm_rotate(x, x, None, i[:4], torch.zeros(9, 64)),
                 lambda: A.prompt_attention(x, x, x, i[:2]),
                 lambda: A.shared_prefix_attention(x, c, c, i, 10, torch.zeros(4, 2, dtype=torch.int32), i[:4])):
        with pytest.raises(VesperError, match="CUDA"):
            call()
