"""The paged-cache, shared-prefix and verification entry points refuse bad calls before any launch: the C
entries with a status and a message (their pointers are never followed), the wrappers with ValueError."""

from __future__ import annotations

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from lazykv_b200 import _lib

    if not _lib.LIB_PATH.exists():
        from lazykv_b200.build import build

        build()
    return _lib.lib()


FIELDS = {
    "PAGED_ARGS": ("keys values k_sb k_st k_sh v_sb v_st v_sh dtype batch tokens h d pages kind scales n_pages bs table table_ld table_cols starts lens "
                   "out_k out_v"),
    "PREFIX_ARGS": ("q dtype q_sb q_st q_sh pages kind scales n_pages bs batch tokens hq h d table table_ld table_cols lens prefix_table prefix_cols "
                    "prefix_len scale out out_dtype lse workspace workspace_bytes"),
    "VERIFY_ARGS": "target p_sb p_st draft q_sb q_st tokens t_sb uniforms u_sb batch k vocab kept token",
}


def _pack(kind: str, fields: dict) -> bytes:
    from lazykv_b200 import _lib

    return getattr(_lib, kind).pack(*[fields[name] for name in FIELDS[kind].split()])


def test_the_packed_structs_have_the_headers_fields() -> None:
    """Names and order of lkv_*_args in include/lkv.h, and the size that a C compiler gives them."""
    import re
    from pathlib import Path

    from lazykv_b200 import _lib

    text = re.sub(r"/\*.*?\*/", "", (Path(__file__).resolve().parents[1] / "include" / "lkv.h").read_text(), flags=re.S)
    sizes = {"int64_t": "q", "int": "i", "float": "f", "size_t": "N"}
    for kind, name in (("PAGED_ARGS", "lkv_paged_args"), ("PREFIX_ARGS", "lkv_prefix_args"), ("VERIFY_ARGS", "lkv_verify_args")):
        body = re.findall(r"typedef struct \{([^}]*)\} %s;" % name, text)[0]
        fields, code = [], "@"
        for line in filter(None, (x.strip() for x in body.split(";"))):
            names = re.sub(r"^(const )?\w+\s*\*?\s*", "", line)
            for f in names.split(","):
                fields.append(f.strip())
                code += "P" if "*" in line else sizes[line.split()[0]]
        assert " ".join(fields) == FIELDS[kind] and code == getattr(_lib, kind).format


def _write(lib, **over: object) -> int:  # noqa: ANN001
    base = dict(keys=4096, values=4096, k_sb=128, k_st=128, k_sh=64, v_sb=128, v_st=128, v_sh=64, dtype=1, batch=2, tokens=1, h=2, d=64, pages=4096, kind=1,
                scales=4096, n_pages=4, bs=16, table=4096, table_ld=3, table_cols=3, starts=4096, lens=0, out_k=0, out_v=0)
    return lib.lkv_paged_write(_pack("PAGED_ARGS", {**base, **over}), None)


@pytest.mark.parametrize("bad,status,message", [
    (dict(dtype=5), 1, "dtype"), (dict(kind=2), 1, "cache kind"), (dict(d=96), 1, "head_dim"), (dict(bs=24), 1, "pages of 24"), (dict(h=0), 1, "bad shape"),
    (dict(batch=-1), 1, "bad shape"), (dict(tokens=-1), 1, "bad shape"), (dict(table_ld=2), 1, "bad shape"), (dict(n_pages=2**31), 1, "bad shape"),
    (dict(batch=2**20, tokens=2**12), 1, "rows"), (dict(scales=0), 2, "null"), (dict(keys=0), 2, "null"), (dict(starts=0), 2, "null"),
    (dict(pages=4104), 2, "16-byte"), (dict(keys=4097), 2, "misaligned"),
])
def test_write_refuses(lib, bad: dict, status: int, message: str) -> None:  # noqa: ANN001
    from lazykv_b200 import _lib

    assert _write(lib, **bad) == status and message in _lib.last_error()


def test_write_of_nothing_is_no_launch(lib) -> None:  # noqa: ANN001
    assert _write(lib, batch=0) == 0 and _write(lib, tokens=0) == 0 and _write(lib, n_pages=0) == 0 and _write(lib, table_cols=0, table_ld=0) == 0
    assert lib.lkv_paged_write(None, None) == 2 and lib.lkv_paged_read(None, None) == 2


def _read(lib, **over: object) -> int:  # noqa: ANN001
    base = dict(keys=0, values=0, k_sb=0, k_st=0, k_sh=0, v_sb=0, v_st=0, v_sh=0, dtype=1, batch=2, tokens=1, h=2, d=64, pages=4096, kind=1, scales=4096,
                n_pages=4, bs=16, table=4096, table_ld=3, table_cols=3, starts=4096, lens=0, out_k=4096, out_v=4096)
    return lib.lkv_paged_read(_pack("PAGED_ARGS", {**base, **over}), None)


@pytest.mark.parametrize("bad,status,message", [
    (dict(dtype=3), 1, "dtype"), (dict(kind=-1), 1, "cache kind"), (dict(d=80), 1, "head_dim"), (dict(bs=256), 1, "pages of 256"), (dict(table_cols=-1), 1, "bad shape"),
    (dict(tokens=2**30), 1, "rows"), (dict(scales=0), 2, "null"), (dict(table=0), 2, "null"), (dict(starts=0), 2, "null"), (dict(out_k=0), 2, "null"),
    (dict(out_v=4104), 2, "16-byte"),
])
def test_read_refuses(lib, bad: dict, status: int, message: str) -> None:  # noqa: ANN001
    from lazykv_b200 import _lib

    assert _read(lib, **bad) == status and message in _lib.last_error()
    assert _read(lib, batch=0) == 0


def _attend(lib, **over: object) -> int:  # noqa: ANN001
    base = dict(q=4096, dtype=1, q_sb=512, q_st=512, q_sh=64, pages=4096, kind=1, scales=4096, n_pages=8, bs=16, batch=2, tokens=1, hq=8, h=2, d=64, table=4096,
                table_ld=3, table_cols=3, lens=4096, prefix_table=4096, prefix_cols=4, prefix_len=60, scale=0.125, out=4096, out_dtype=1, lse=4096,
                workspace=4096, workspace_bytes=1 << 30)
    return lib.lkv_prefix_attention(_pack("PREFIX_ARGS", {**base, **over}), None)


@pytest.mark.parametrize("bad,status,message", [
    (dict(kind=4), 1, "cache kind"), (dict(dtype=0), 1, "dtype"), (dict(out_dtype=9), 1, "dtype"), (dict(d=32), 1, "head_dim"), (dict(bs=8), 1, "pages of 8"),
    (dict(hq=7), 1, "do not group"), (dict(h=0), 1, "do not group"), (dict(batch=-2), 1, "bad shape"), (dict(table_ld=2), 1, "bad shape"),
    (dict(prefix_len=-1), 1, "bad shape"), (dict(prefix_len=65), 1, "a prefix of 65"), (dict(batch=70000), 1, "a batch of 70000"),
    (dict(tokens=2**23, batch=1), 1, "a batch of 1"), (dict(table_cols=2**28, table_ld=2**28), 1, "2^30"), (dict(batch=60000, h=60000, hq=60000), 1, "row tiles"), (dict(q=0), 2, "null"), (dict(lens=0), 2, "null"),
    (dict(scales=0), 2, "null"), (dict(prefix_table=0), 2, "null"), (dict(out=0), 2, "null"), (dict(lse=0), 2, "null"),
    (dict(q=4104), 2, "aligned"), (dict(q_sh=68), 2, "aligned"), (dict(workspace_bytes=64), 4, "workspace"), (dict(workspace=0), 2, "workspace"),
])
def test_attention_refuses(lib, bad: dict, status: int, message: str) -> None:  # noqa: ANN001
    from lazykv_b200 import _lib

    assert _attend(lib, **bad) == status and message in _lib.last_error()


def test_attention_of_nothing_and_its_workspace(lib) -> None:  # noqa: ANN001
    from lazykv_b200 import _lib

    assert lib.lkv_prefix_attention(None, None) == 2 and "null" in _lib.last_error()
    assert _attend(lib, batch=0) == 0
    assert _attend(lib, tokens=0) == 0
    assert lib.lkv_prefix_attention_workspace(4, 1, 32, 8, 128, 0, 0, 0) == 0  # nothing to attend, no partials
    one = lib.lkv_prefix_attention_workspace(4, 1, 32, 8, 128, 1, 0, 0)
    assert one >= 4 * 32 * (128 * 4 + 8)
    assert lib.lkv_prefix_attention_workspace(4, 1, 32, 8, 128, 1, 0, 1000) > one
    assert lib.lkv_prefix_attention_workspace(4, 1, 32, 8, 128, 100_000, 0, 0) > one


def _verify(lib, **over: object) -> int:  # noqa: ANN001
    base = dict(target=4096, p_sb=400, p_st=100, draft=4096, q_sb=300, q_st=100, tokens=4096, t_sb=3, uniforms=4096, u_sb=4, batch=2, k=3, vocab=100, kept=4096,
                token=4096)
    return lib.lkv_verify_drafts(_pack("VERIFY_ARGS", {**base, **over}), None)


@pytest.mark.parametrize("bad,status,message", [
    (dict(batch=-1), 1, "bad shape"), (dict(k=-1), 1, "bad shape"), (dict(vocab=0), 1, "bad shape"), (dict(vocab=2**22 + 1), 1, "bad shape"),
    (dict(target=0), 2, "null"), (dict(tokens=0), 2, "null"), (dict(uniforms=0), 2, "null"), (dict(kept=0), 2, "null"), (dict(token=0), 2, "null"),
    (dict(target=4098), 2, "misaligned"), (dict(tokens=4100), 2, "misaligned"),
])
def test_verification_refuses(lib, bad: dict, status: int, message: str) -> None:  # noqa: ANN001
    from lazykv_b200 import _lib

    assert _verify(lib, **bad) == status and message in _lib.last_error()
    assert _verify(lib, batch=0) == 0 and lib.lkv_verify_drafts(None, None) == 2


def test_the_wrappers_take_cuda_tensors_only() -> None:
    from lazykv_b200 import kernels as K

    x, ints = torch.zeros((1, 1, 2, 64)), torch.zeros(1, dtype=torch.int32)
    pages, table = torch.zeros((1, 2, 2, 16, 64)), torch.zeros((1, 1), dtype=torch.int32)
    for call in (lambda: K.paged_write(x, x, pages, table, ints), lambda: K.paged_read(pages, table, ints, 1),
                 lambda: K.prefix_attention(x.bfloat16(), pages, table, ints, table[0], 1, 1.0),
                 lambda: K.verify_drafts(torch.zeros((1, 2, 3)), None, torch.zeros((1, 1), dtype=torch.int64), torch.zeros((1, 2)))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
