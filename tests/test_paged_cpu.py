"""The paged-cache, shared-prefix and verification entry points refuse bad calls before any launch: the C
entries with a status and a message (their pointers are never followed), the wrappers with ValueError."""

from __future__ import annotations

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from lazykv_b200 import _lib

    if not _lib.LIB_PATH.exists():
        from lazykv_b200.build import build

        build()
    return _lib.lib()


FAKE = ctypes.c_void_p(4096)


def _write(lib, keys=FAKE, dtype=1, batch=2, tokens=1, h=2, d=64, pages=FAKE, kind=1, scales=FAKE, n_pages=4, bs=16, ld=3, cols=3, starts=FAKE):  # noqa: ANN001, ANN202
    return lib.lkv_paged_write(keys, 128, 128, 64, FAKE, 128, 128, 64, dtype, batch, tokens, h, d, pages, kind, scales, n_pages, bs, FAKE, ld, cols, starts, None)


@pytest.mark.parametrize("bad,status,message", [
    (dict(dtype=5), 1, "dtype"), (dict(kind=2), 1, "cache kind"), (dict(d=96), 1, "head_dim"), (dict(bs=24), 1, "pages of 24"), (dict(h=0), 1, "bad shape"),
    (dict(batch=-1), 1, "bad shape"), (dict(tokens=-1), 1, "bad shape"), (dict(ld=2), 1, "bad shape"), (dict(n_pages=2**31), 1, "bad shape"),
    (dict(batch=2**20, tokens=2**12), 1, "rows"), (dict(scales=None), 2, "null"), (dict(keys=None), 2, "null"), (dict(starts=None), 2, "null"),
    (dict(pages=ctypes.c_void_p(4104)), 2, "16-byte"), (dict(keys=ctypes.c_void_p(4097)), 2, "misaligned"),
])
def test_write_refuses(lib, bad: dict, status: int, message: str) -> None:  # noqa: ANN001
    from lazykv_b200 import _lib

    assert _write(lib, **bad) == status and message in _lib.last_error()


def test_write_of_nothing_is_no_launch(lib) -> None:  # noqa: ANN001
    assert _write(lib, batch=0) == 0 and _write(lib, tokens=0) == 0 and _write(lib, n_pages=0) == 0 and _write(lib, cols=0, ld=0) == 0


def _read(lib, dtype=1, batch=2, tokens=1, h=2, d=64, pages=FAKE, kind=1, scales=FAKE, bs=16, ld=3, cols=3, table=FAKE, starts=FAKE, out=FAKE):  # noqa: ANN001, ANN202
    return lib.lkv_paged_read(pages, kind, scales, 4, bs, batch, tokens, h, d, table, ld, cols, starts, None, out, FAKE, dtype, None)


@pytest.mark.parametrize("bad,status,message", [
    (dict(dtype=3), 1, "dtype"), (dict(kind=-1), 1, "cache kind"), (dict(d=80), 1, "head_dim"), (dict(bs=256), 1, "pages of 256"), (dict(cols=-1), 1, "bad shape"),
    (dict(tokens=2**30), 1, "rows"), (dict(scales=None), 2, "null"), (dict(table=None), 2, "null"), (dict(starts=None), 2, "null"), (dict(out=None), 2, "null"),
    (dict(out=ctypes.c_void_p(4104)), 2, "16-byte"),
])
def test_read_refuses(lib, bad: dict, status: int, message: str) -> None:  # noqa: ANN001
    from lazykv_b200 import _lib

    assert _read(lib, **bad) == status and message in _lib.last_error()
    assert _read(lib, batch=0) == 0


def _args(**over: object):  # noqa: ANN202
    from lazykv_b200 import _lib

    a = _lib.PrefixArgs()
    base = dict(q=4096, dtype=1, q_sb=512, q_st=512, q_sh=64, pages=4096, kind=1, scales=4096, n_pages=8, bs=16, batch=2, tokens=1, hq=8, h=2, d=64, table=4096,
                table_ld=3, table_cols=3, lens=4096, prefix_table=4096, prefix_cols=4, prefix_len=60, scale=0.125, out=4096, out_dtype=1, lse=4096,
                workspace=4096, workspace_bytes=1 << 30)
    for k, v in {**base, **over}.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad,status,message", [
    (dict(kind=4), 1, "cache kind"), (dict(dtype=0), 1, "dtype"), (dict(out_dtype=9), 1, "dtype"), (dict(d=32), 1, "head_dim"), (dict(bs=8), 1, "pages of 8"),
    (dict(hq=7), 1, "do not group"), (dict(h=0), 1, "do not group"), (dict(batch=-2), 1, "bad shape"), (dict(table_ld=2), 1, "bad shape"),
    (dict(prefix_len=-1), 1, "bad shape"), (dict(prefix_len=65), 1, "a prefix of 65"), (dict(batch=70000), 1, "a batch of 70000"),
    (dict(tokens=2**23, batch=1), 1, "a batch of 1"), (dict(table_cols=2**28, table_ld=2**28), 1, "2^30"), (dict(q=None), 2, "null"), (dict(lens=None), 2, "null"),
    (dict(scales=None), 2, "null"), (dict(prefix_table=None), 2, "null"), (dict(out=None), 2, "null"), (dict(lse=None), 2, "null"),
    (dict(q=4104), 2, "aligned"), (dict(q_sh=68), 2, "aligned"), (dict(workspace_bytes=64), 4, "workspace"), (dict(workspace=None), 2, "workspace"),
])
def test_attention_refuses(lib, bad: dict, status: int, message: str) -> None:  # noqa: ANN001
    from lazykv_b200 import _lib

    a = _args(**bad)
    assert lib.lkv_prefix_attention(ctypes.byref(a), None) == status and message in _lib.last_error()


def test_attention_of_nothing_and_its_workspace(lib) -> None:  # noqa: ANN001
    from lazykv_b200 import _lib

    assert lib.lkv_prefix_attention(None, None) == 2 and "null" in _lib.last_error()
    assert lib.lkv_prefix_attention(ctypes.byref(_args(batch=0)), None) == 0
    assert lib.lkv_prefix_attention(ctypes.byref(_args(tokens=0)), None) == 0
    assert lib.lkv_prefix_attention_workspace(4, 1, 32, 8, 128, 0, 0, 0) == 0  # nothing to attend, no partials
    one = lib.lkv_prefix_attention_workspace(4, 1, 32, 8, 128, 1, 0, 0)
    assert one >= 4 * 32 * (128 * 4 + 8)
    assert lib.lkv_prefix_attention_workspace(4, 1, 32, 8, 128, 1, 0, 1000) > one
    assert lib.lkv_prefix_attention_workspace(4, 1, 32, 8, 128, 100_000, 0, 0) > one


def _verify(lib, target=FAKE, tokens=FAKE, uniforms=FAKE, batch=2, k=3, vocab=100, kept=FAKE, token=FAKE):  # noqa: ANN001, ANN202
    return lib.lkv_verify_drafts(target, 400, 100, FAKE, 300, 100, tokens, 3, uniforms, 4, batch, k, vocab, kept, token, None)


@pytest.mark.parametrize("bad,status,message", [
    (dict(batch=-1), 1, "bad shape"), (dict(k=-1), 1, "bad shape"), (dict(vocab=0), 1, "bad shape"), (dict(vocab=2**22 + 1), 1, "bad shape"),
    (dict(target=None), 2, "null"), (dict(tokens=None), 2, "null"), (dict(uniforms=None), 2, "null"), (dict(kept=None), 2, "null"), (dict(token=None), 2, "null"),
    (dict(target=ctypes.c_void_p(4098)), 2, "misaligned"), (dict(tokens=ctypes.c_void_p(4100)), 2, "misaligned"),
])
def test_verification_refuses(lib, bad: dict, status: int, message: str) -> None:  # noqa: ANN001
    from lazykv_b200 import _lib

    assert _verify(lib, **bad) == status and message in _lib.last_error()
    assert _verify(lib, batch=0) == 0


def test_the_wrappers_take_cuda_tensors_only() -> None:
    from lazykv_b200 import kernels as K

    x, ints = torch.zeros((1, 1, 2, 64)), torch.zeros(1, dtype=torch.int32)
    pages, table = torch.zeros((1, 2, 2, 16, 64)), torch.zeros((1, 1), dtype=torch.int32)
    for call in (lambda: K.paged_write(x, x, pages, table, ints), lambda: K.paged_read(pages, table, ints, 1),
                 lambda: K.prefix_attention(x.bfloat16(), pages, table, ints, table[0], 1, 1.0),
                 lambda: K.verify_drafts(torch.zeros((1, 2, 3)), None, torch.zeros((1, 1), dtype=torch.int64), torch.zeros((1, 2)))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
