"""The operators around an expert layer's products, and dropout: what the sources and the header say - what cannot be seen
from results on a device without a misuse there, and what a C or C++ program meets."""
import os
import re
import shutil
import subprocess

import pytest

from test_dependent_launch import _functions, _source

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_places_out_of_memory_are_bounded_before_a_store():
    """dispatch's copies store a row where a number out of memory says.  What is not below the number of slots is skipped:
    executions that share a scratchpad against the rules may make any number."""
    functions = _functions(_source("moe_dispatch.cu"))
    copy, shift = functions["dispatch_copy_kernel"], functions["dispatch_shift_kernel"]
    assert re.search(r"slots = \(uint32_t\)a\.tokens \* a\.choices;", copy)
    assert re.search(r"if \(\(uint32_t\)to\[q\]\[j\] < slots\) \*\(uint4 \*\)", copy)
    assert re.search(r"if \(\(uint32_t\)mine >= \(uint32_t\)a\.tokens \* a\.choices\) mine = -1;", shift)
    assert re.search(r"to = __shfl_sync\(0xffffffffu, mine, j\);\s*if \(to < 0\) continue;", shift)
    assert "max(kept, 0)" in functions["zero_behind"]


NAMES = ["SRC", "SRC_1", "SRC_2", "DST", "DST_1", "WEIGHTS", "DIFF_SRC", "DIFF_DST", "DIFF_WEIGHTS", "ATTR_DROPOUT_SEED"]
# as oneDNN's dnnl_types.h documents them
NUMBERS = [1, 2, 3, 17, 18, 33, 129, 145, 161, 511]


def argument_ids(tmp_path, first=None, include=()):
    """the ids a C++ program sees that includes `first` and then this library's header"""
    source = "".join('#include "%s"\n' % h for h in ([first] if first else []) + ["dnnl_b200.h"])
    source += "#include <stdio.h>\nint main() {" + "".join('printf("%%d ", DNNL_ARG_%s);' % n for n in NAMES) + " return 0; }\n"
    (tmp_path / "ids.cpp").write_text(source)
    exe = str(tmp_path / "ids")
    r = subprocess.run([shutil.which("g++") or "/usr/bin/g++", "-std=c++17", str(tmp_path / "ids.cpp"), "-I" + os.path.join(ROOT, "include"), "-o", exe]
                       + ["-I" + i for i in include], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
    return [int(v) for v in subprocess.run([exe], capture_output=True, text=True, timeout=60).stdout.split()]


def test_argument_ids_are_those_of_the_reference(tmp_path, host_engine):
    """a program that includes oneDNN's own header first gets its numbers for these arguments, and the library has to know
    a tensor by them"""
    from onednn_b200 import api
    assert [getattr(api, "ARG_" + n) for n in NAMES] == NUMBERS
    assert argument_ids(tmp_path) == NUMBERS
    m = api.memory.desc((5, 4), 3, (4, 1))
    pd = api.dropout.primitive_desc(host_engine, m, m, 0.5)
    assert pd.query_md(255, 511) == api.memory.desc((2,), 16, (1,)) and pd.query_md(255, 510).get_ndims() == 0


def test_argument_ids_behind_the_reference_header(tmp_path):
    import torch
    include = os.path.join(os.path.dirname(torch.__file__), "include")
    if not os.path.exists(os.path.join(include, "oneapi", "dnnl", "dnnl.h")):
        pytest.skip("no oneDNN header on this machine")
    assert argument_ids(tmp_path, "oneapi/dnnl/dnnl.h", [include]) == NUMBERS


def test_kinds_outside_the_reference_enum_are_numbers(host_engine):
    """dnnl_primitive_kind_t ends at 0x7fff; a C++ enum object may not hold the kinds of this library's own primitives"""
    import ctypes as C

    from onednn_b200 import api
    sources = os.path.join(ROOT, "onednn_b200", "csrc")
    for f in sorted(os.listdir(sources)):
        if f.endswith((".cu", ".hpp", ".h", ".cuh")):
            assert not re.search(r"\(dnnl_primitive_kind_t\s*\*?\)", open(os.path.join(sources, f)).read()), f
    assert re.search(r"struct dnnl_primitive_desc \{[^}]*\n    int kind = dnnl_matmul;", _source("objects.hpp"))
    lib, m, kind = api.lib(), api.memory.desc((5, 4), 3, (4, 1)), C.c_int()
    pd = api.dropout.primitive_desc(host_engine, m, m, 0.5)
    assert lib.dnnl_primitive_desc_query(pd._h, 2, 0, C.byref(kind)) == 0 and kind.value == 0x10006
    lib.dnnl_prim_kind2str.restype = C.c_char_p
    assert [lib.dnnl_prim_kind2str(k) for k in (0x10006, 0x10001, 0x10007, 14, 1)] == [
        b"dropout", b"moe_route", b"unknown prim_kind", b"matmul", b"reorder"]


def test_the_example_compares_every_gradient_that_it_makes():
    """examples/moe_layer.py: what the steps of its way back write is what run() compares with plain torch"""
    text = open(os.path.join(ROOT, "examples", "moe_layer.py")).read()
    steps = re.search(r"def backward\(self\):\s*for step in \(([^)]*)\)", text).group(1)
    written = set()
    for step in re.findall(r"self\.(\w+)", steps):
        body = re.search(r"s = self\.%s = Step\(self\)(.*?)\n\n" % step, text, re.S).group(1)
        written |= set(re.findall(r"api\.ARG_(?:DST|DIFF_SRC|DIFF_WEIGHTS), self\.(\w+)\)", body))
    compared = re.search(r"results = \{(.*?)\}\n", text).group(1)
    assert written == {"drows", "dw", "dlogits"}
    assert all("layer." + name in compared for name in written)


def test_an_empty_matrix_may_have_any_strides(host_engine):
    """tensor libraries give matrices without elements strides of zero"""
    from onednn_b200 import api
    md, O = api.memory.desc, api.RUNTIME_DIM_VAL
    f, i = md((0, 2), 3, (0, 0)), md((0, 2), 4, (0, 0))
    rows = md.grouped((0, 4), 3, 0, 8)
    api.moe_route.primitive_desc(host_engine, md((0, 8), 3, (0, 0)), f, i)
    api.moe_dispatch.primitive_desc(host_engine, md((0, 4), 3, (0, 0)), i, rows, i)
    api.moe_combine.primitive_desc(host_engine, rows, i, md((0, 4), 3, (0, 0)), weights_md=f)
    api.dropout.primitive_desc(host_engine, md((5, 0), 3, (0, 0)), md((5, 0), 3, (0, 0)), 0.5)
    with pytest.raises(api.error) as e:  # but a known pitch of outputs with rows still counts
        api.dropout.primitive_desc(host_engine, md((5, 4), 3, (4, 1)), md((5, 4), 3, (0, 1)), 0.5)
    assert e.value.status == api.unimplemented


@pytest.mark.parametrize("file", ["sm100_ptx.cuh", "token_rows.cuh", "moe_route.cu", "moe_dispatch.cu", "moe_combine.cu", "dropout.cu"])
def test_every_function_is_called(file):
    sources = os.path.join(ROOT, "onednn_b200", "csrc")
    text = "".join(_source(f) for f in os.listdir(sources) if f.endswith((".cu", ".cuh", ".h", ".hpp")))
    assert not [n for n in _functions(_source(file)) if len(re.findall(r"\b%s\b" % n, text)) < 2]
