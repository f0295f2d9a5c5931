"""What the packed-chunk operators refuse, before anything touches a device."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from lazykv_b200 import _lib as L

FAKE = 4096  # never dereferenced: every call below fails its checks first


@pytest.fixture(scope="module")
def lib():  # noqa: ANN201
    if not L.LIB_PATH.exists():
        from lazykv_b200.build import build

        build()
    return L.lib()


def _fields(layout, base: dict, names: list[str]):  # noqa: ANN001, ANN202
    def make(**change):  # noqa: ANN003, ANN202
        return layout.pack(*[{**base, **change}[n] for n in names])

    return make


ROTATE = ["q", "k", "v", "q_st", "q_sh", "k_st", "k_sh", "v_st", "v_sh", "out", "o_st", "o_sh", "dtype", "rows", "hq", "h", "d", "positions", "frequencies", "pairs",
          "interleaved", "qw", "kw", "eps", "pages", "kind", "scales", "n_pages", "bs", "table", "ld", "cols", "lens", "offsets", "batch"]
EVICT = ["pages", "kind", "dtype", "scales", "n_pages", "h", "bs", "d", "batch", "table", "ld", "cols", "lens", "sums", "positions", "cap", "out_sums", "out_positions", "out_lens",
         "keep", "sinks", "since", "workspace", "workspace_bytes"]
CHUNK = ["q", "q_st", "q_sh", "dtype", "rows", "hq", "h", "d", "pages", "kind", "scales", "n_pages", "bs", "table", "ld", "cols", "lens", "offsets", "batch", "prefix_table",
         "prefix_cols", "prefix_len", "scale", "cap", "out", "lse", "workspace", "workspace_bytes"]
SUMS = ["q", "q_st", "q_sh", "dtype", "rows", "hq", "h", "d", "lse", "pages", "kind", "scales", "n_pages", "bs", "table", "ld", "cols", "lens", "offsets", "batch", "last", "sums",
        "out", "cap", "scale", "cap_scores", "workspace", "workspace_bytes"]
BASE = {"q": FAKE, "k": FAKE, "v": FAKE, "q_st": 512, "q_sh": 64, "k_st": 128, "k_sh": 64, "v_st": 128, "v_sh": 64, "out": FAKE, "o_st": 512, "o_sh": 64, "dtype": 1, "rows": 9, "hq": 8,
        "h": 2, "d": 64, "positions": FAKE, "frequencies": FAKE, "pairs": 32, "interleaved": 0, "qw": 0, "kw": 0, "eps": 1e-6, "pages": FAKE, "kind": 0, "scales": 0, "n_pages": 10,
        "bs": 16, "table": FAKE, "ld": 3, "cols": 3, "lens": FAKE, "offsets": FAKE, "batch": 2, "sums": FAKE, "cap": 48, "out_sums": FAKE, "out_positions": FAKE, "out_lens": 2 * FAKE,
        "keep": 10, "sinks": 0, "since": 0, "workspace": FAKE, "workspace_bytes": 1 << 30, "prefix_table": FAKE, "prefix_cols": 2, "prefix_len": 20, "scale": 0.125, "lse": FAKE,
        "last": 100, "cap_scores": 0.0}


@pytest.mark.parametrize(("entry", "layout", "names", "more", "bad"), [
    ("lkv_paged_write_rotated", L.ROTATE_ARGS, ROTATE, {}, [
        ({"d": 96}, 1, "head_dim"), ({"bs": 24}, 1, "pages of 24"), ({"dtype": 5}, 1, "dtype"), ({"pairs": 6}, 1, "rotated pairs"), ({"pairs": 36}, 1, "rotated pairs"),
        ({"rows": -1}, 1, "bad shape"), ({"ld": 2}, 1, "bad shape"), ({"eps": math.nan}, 1, "eps"), ({"q": 0}, 2, "null"), ({"positions": 0}, 2, "null"), ({"k": FAKE + 1}, 2, "misaligned"),
        ({"kind": 1}, 2, "null"), ({"pages": FAKE + 8}, 2, "16-byte")]),
    ("lkv_paged_evict", L.EVICT_ARGS, EVICT, {}, [
        ({"keep": 0}, 1, "budget"), ({"cap": -1}, 1, "bad shape"), ({"out_lens": FAKE}, 2, "in place"), ({"sums": 0}, 2, "null"), ({"workspace_bytes": 8}, 4, "needed"),
        ({"kind": 7}, 1, "cache kind"), ({"h": 0}, 1, "bad shape")]),
    ("lkv_chunk_attention", L.CHUNK_ARGS, CHUNK, {"cap": 0.0}, [
        ({"dtype": 0}, 1, "bfloat16"), ({"hq": 7}, 1, "query heads"), ({"batch": 9000}, 1, "at most"), ({"prefix_len": 33}, 1, "prefix of 33"), ({"cap": -1.0}, 1, "cap"),
        ({"cap": math.inf}, 1, "cap"), ({"scale": math.nan}, 1, "scale"), ({"q": FAKE + 2}, 2, "16-byte"), ({"q_st": 516}, 2, "16-byte"), ({"workspace": 0}, 4, "needed"),
        ({"workspace_bytes": 100}, 4, "needed"), ({"prefix_table": 0}, 2, "null"), ({"n_pages": 2**30}, 1, "rows of pages")]),
    ("lkv_attention_sums", L.SUMS_ARGS, SUMS, {}, [
        ({"last": 0}, 1, "last"), ({"hq": 5}, 1, "query heads"), ({"cap_scores": -2.0}, 1, "cap"), ({"lse": 0}, 2, "null"), ({"out": 0}, 2, "null"), ({"workspace_bytes": 0}, 4, "needed"),
        ({"cap": 2**30 + 1}, 1, "bad shape"), ({"q_sh": 60}, 2, "16-byte"), ({"kind": 1, "scales": FAKE + 4}, 2, "scales must be 16-byte")]),
])
def test_entries_refuse(lib, entry, layout, names, more, bad) -> None:  # noqa: ANN001
    make = _fields(layout, {**BASE, **more}, names)
    call = getattr(lib, entry)
    assert call(None, None) == 2 and "null arguments" in L.last_error()
    for change, code, says in bad:
        assert call(make(**change), None) == code, (change, L.last_error())
        assert says in L.last_error() and entry in L.last_error(), (change, L.last_error())
    empty = {"rows": 0} if "rows" in names and entry != "lkv_attention_sums" else {"batch": 0}
    assert call(make(**empty), None) == 0  # nothing to do


def test_struct_layouts_match_the_header(tmp_path) -> None:  # noqa: ANN001
    import shutil
    import subprocess
    from pathlib import Path

    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    root = Path(__file__).resolve().parents[1]
    names = {"lkv_rotate_args": L.ROTATE_ARGS, "lkv_evict_args": L.EVICT_ARGS, "lkv_chunk_args": L.CHUNK_ARGS, "lkv_sums_args": L.SUMS_ARGS}
    src = '#include <stdio.h>\n#include "lkv.h"\nint main(void) {' + "".join(f'printf("%zu ", sizeof({n}));' for n in names) + "return 0; }\n"
    (tmp_path / "t.c").write_text(src)
    subprocess.run(["gcc", "-I", str(root / "include"), str(tmp_path / "t.c"), "-o", str(tmp_path / "t")], check=True)
    sizes = [int(x) for x in subprocess.check_output([str(tmp_path / "t")]).split()]
    for size, (name, layout) in zip(sizes, names.items()):
        assert size == -(-layout.size // 8) * 8, name  # (a struct's size is a multiple of its alignment)


def test_workspaces(lib) -> None:  # noqa: ANN001
    assert lib.lkv_paged_evict_workspace(2, 3, 100, 30) == 2 * 3 * 30 * 8
    assert lib.lkv_paged_evict_workspace(2, 3, 100, 80) == 2 * 3 * 20 * 8
    assert lib.lkv_paged_evict_workspace(2, 3, 100, 100) == 0
    assert lib.lkv_chunk_attention_workspace(0, 2, 8, 2, 64, 0, 48) == 0
    small, most = lib.lkv_chunk_attention_workspace(1, 1, 1, 1, 64, 0, 16), lib.lkv_chunk_attention_workspace(1 << 20, 64, 32, 8, 128, 0, 1 << 20)
    assert 0 < small < most <= 2 * 148 * (256 * 128 * 4 + 256 * 8 + 16)
    assert 0 < lib.lkv_attention_sums_workspace(1, 1, 16) <= lib.lkv_attention_sums_workspace(64, 8, 4096) <= 2 * 148 * (1024 + 16)


def test_debug_hooks_are_bounded(lib) -> None:  # noqa: ANN001
    assert lib.lkv_debug_set(L.LKV_DEBUG_CHUNK_WAIT_NS, ctypes.c_int64(0)) == 1 and "chunk wait bound" in L.last_error()
    assert lib.lkv_debug_set(L.LKV_DEBUG_CHUNK_STALL_NEXT, ctypes.c_int64(3)) == 1 and "no stall 3" in L.last_error()


def test_wrappers_take_cuda_tensors_only() -> None:
    from lazykv_b200 import kernels as K

    q, k, i = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32)
    pages, table = torch.zeros(2, 2, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda: K.paged_write_rotated(q, k, k, i, torch.zeros(4), pages, table, i[:1], i[:2]),
                 lambda: K.chunk_attention(q, pages, table, i[:1], i[:2], 1.0),
                 lambda: K.attention_sums(q, torch.zeros(3, 4), pages, table, i[:1], i[:2], 1.0),
                 lambda: K.paged_evict(pages, table, i[:1], torch.zeros(1, 2, 32), torch.zeros(1, 2, 32, dtype=torch.int32), 4)):
        with pytest.raises(ValueError, match="no CPU fallback"):
            call()
