"""The digest that ties profiles of encode_img to its kernels (lib.source_digest): another path's kernel does not orphan them, their own does."""
import os
import shutil

import pytest

from hawkeye_amd import lib as L

CSRC = os.path.join(os.path.dirname(os.path.abspath(L.__file__)), "csrc")


@pytest.fixture
def csrc(tmp_path):
    for name in os.listdir(CSRC):
        if name.endswith((".hip", ".h")) or name == "Makefile":
            shutil.copy(os.path.join(CSRC, name), tmp_path)
    assert L.source_digest(str(tmp_path)) == L.source_digest()
    return tmp_path


def _edit(path, old, new):
    text = path.read_text()
    assert old in text
    path.write_text(text.replace(old, new, 1))


def test_other_paths_and_comments_leave_the_digest_alone(csrc):
    for name in ("hk_attn_prefix.hip", "hk_cache.hip", "hk_decode.hip", "hk_llm.hip", "hk_train.hip", "hk_attn_causal.hip", "hk_overlap.h"):
        with open(csrc / name, "a") as f:
            f.write("\nstatic int one_more_function() { return 1; }\n")
    (csrc / "hk_new_operator.hip").write_text("int x;\n")
    with open(csrc / "hk_gemm.hip", "a") as f:
        f.write("\n// a note\n/* and another */\n")
    _edit(csrc / "Makefile", "SRCS = ", "SRCS = hk_new_operator.hip ")
    assert L.source_digest(str(csrc)) == L.source_digest()


@pytest.mark.parametrize("name", L.ENCODE_SOURCES)
def test_the_paths_own_sources_change_it(csrc, name):
    with open(csrc / name, "a") as f:
        f.write("\nstatic int one_more_function() { return 1; }\n")
    assert L.source_digest(str(csrc)) != L.source_digest()


@pytest.mark.parametrize("old,new", [("-O3", "-O2"), ("-Xclang -packed-fp32-ops", ""), ("-fno-honor-nans -fno-slp-vectorize", "-fno-honor-nans")])
def test_the_flags_they_are_compiled_with_change_it(csrc, old, new):
    _edit(csrc / "Makefile", old, new)
    assert L.source_digest(str(csrc)) != L.source_digest()


def test_the_sources_are_those_of_the_entry_points_the_engine_calls():
    import re
    engine = open(os.path.join(os.path.dirname(CSRC), "engine.py")).read()
    used = set(re.findall(r"lib\.(hk_\w+)", engine)) | {"hk_cast_f32_bf16", "hk_pos_embed"}
    for fn in used:
        where = [n for n in os.listdir(CSRC) if n.endswith(".hip") and re.search(r'extern "C" \w+ %s\(' % fn, open(os.path.join(CSRC, n)).read())]
        assert len(where) == 1 and where[0] in L.ENCODE_SOURCES, (fn, where)
