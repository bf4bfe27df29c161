"""CPU tests of the training entry points: the C structure's layout and every refusal."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import flash_mlm
from flash_mlm import _lib
from flash_mlm.host.cache import PackMetadata

ROOT = Path(__file__).resolve().parents[1]
F16 = torch.float16


@pytest.mark.skipif(shutil.which("gcc") is None and shutil.which("cc") is None, reason="no C compiler")
def test_backward_args_match_header(tmp_path):
    cls, cname = _lib.AttnBwdArgs, "fmlm_attn_bwd_args"
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "flash_mlm.h"', "int main(void) {",
             f'  printf("sizeof %zu\\n", sizeof({cname}));']
    lines += [f'  printf("{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "abi.c", tmp_path / "abi"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run([shutil.which("gcc") or shutil.which("cc"), "-std=c11", "-I", str(ROOT / "include"), str(src), "-o",
                    str(exe)], check=True)
    got = dict(x.split() for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert int(got["sizeof"]) == ctypes.sizeof(cls)
    for f, _ in cls._fields_:
        assert int(got[f]) == getattr(cls, f).offset, f


def meta(lens, N):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    i32 = dict(dtype=torch.int32)
    return PackMetadata(B=len(lens), N=N, lengths=torch.tensor(lens, **i32), cu_seqlens=torch.tensor(cu, **i32),
                        token_indices=torch.zeros(cu[-1], dtype=torch.int64), total_tokens=cu[-1], batch_ids_block_n=64,
                        batch_ids_q=torch.zeros(0, **i32), q_tile_starts_q=torch.zeros(0, **i32))


def z(*shape, dtype=F16):
    return torch.zeros(shape, dtype=dtype)


REFUSED = [
    ("rank", dict(q=z(4, 64)), "rank-4"),
    ("ranks differ", dict(q=z(2, 4, 8, 64), k=z(4, 8, 64), v=z(4, 8, 64)), "rank-4"),
    ("k and v", dict(v=z(2, 4, 8, 32)), "same shape"),
    ("lengths differ", dict(k=z(2, 4, 9, 64), v=z(2, 4, 9, 64)), "heads only"),
    ("batch differs", dict(k=z(3, 4, 8, 64), v=z(3, 4, 8, 64)), "heads only"),
    ("heads", dict(k=z(2, 3, 8, 64), v=z(2, 3, 8, 64)), "multiple"),
    ("head_dim", dict(q=z(2, 4, 8, 48), k=z(2, 4, 8, 48), v=z(2, 4, 8, 48)), "HEAD_DIM"),
    ("dtype", dict(q=z(2, 4, 8, 64, dtype=torch.float32), k=z(2, 4, 8, 64, dtype=torch.float32),
                   v=z(2, 4, 8, 64, dtype=torch.float32)), "dtype"),
    ("dtypes differ", dict(k=z(2, 4, 8, 64, dtype=torch.bfloat16)), "same dtype"),
    ("packed without meta", dict(q=z(4, 8, 64), k=z(4, 8, 64), v=z(4, 8, 64)), "q_meta"),
    ("packed count", dict(q=z(4, 8, 64), k=z(4, 8, 64), v=z(4, 8, 64), q_meta=meta([3, 4], 8)), "token count"),
    ("padded meta", dict(q_meta=meta([3, 4], 9)), "padded shape"),
    ("context in part", dict(q_meta=meta([3, 4], 8), context_k=z(4, 5, 64)), "together"),
    ("context without meta", dict(context_k=z(4, 5, 64), context_v=z(4, 5, 64), context_meta=meta([5], 5)), "q_meta"),
    ("causal without meta", dict(causal_query_seq_attn=True), "q_meta"),
    ("context shape", dict(q_meta=meta([3, 4], 8), context_k=z(4, 6, 64), context_v=z(4, 6, 64), context_meta=meta([5], 5)),
     "context_k and context_v must be"),
    ("context entries", dict(q_meta=meta([3, 4], 8), context_k=z(4, 5, 64), context_v=z(4, 5, 64),
                             context_meta=meta([1, 2, 2], 5)), "one context"),
    ("cpu", dict(), "CUDA"),
]


@pytest.mark.parametrize("what,change,message", REFUSED, ids=[r[0] for r in REFUSED])
@pytest.mark.parametrize("entry", ["fwd", "bwd", "train"])
def test_refusals(what, change, message, entry):
    kw = dict(q=z(2, 4, 8, 64), k=z(2, 4, 8, 64), v=z(2, 4, 8, 64), scale=0.125)
    kw.update(change)
    if entry == "bwd":
        kw.update(dout=kw["q"], out=kw["q"], lse=torch.zeros(kw["q"].shape[:-1]))
    with pytest.raises(ValueError, match=message):
        getattr(flash_mlm, f"flash_attn_mlm_{entry}")(**kw)


def bwd_args(**change):
    """A well-formed packed argument block over made-up addresses (never launched: each test breaks one field)."""
    a = _lib.AttnBwdArgs()
    a.dtype, a.head_dim, a.layout, a.batch, a.num_heads, a.kv_heads = 1, 64, _lib.FMLM_BWD_PACKED, 2, 4, 2
    a.scale, a.total_q_len = 0.125, 10

    def view(heads):
        return _lib.View4(1 << 20, 10, heads, 1, 64, 640, 640 * heads)

    a.q, a.dout, a.k, a.v = view(4), view(4), view(2), view(2)
    for f in ("out", "lse", "cu_seqlens_q", "dq", "dk", "dv", "workspace", "error_word"):
        setattr(a, f, 1 << 20)
    a.workspace_bytes = 1 << 16
    for f, x in change.items():
        setattr(a, f, x)
    return a


@pytest.mark.parametrize("change,message", [
    (dict(dtype=2), "dtype"), (dict(layout=3), "layout"), (dict(batch=0), "batch"), (dict(kv_heads=3), "multiple"),
    (dict(total_q_len=0), "total_q_len"), (dict(total_q_len=1 << 30), "total_q_len"),
    (dict(layout=_lib.FMLM_BWD_DENSE), "seq_len"), (dict(cu_seqlens_q=None), "cu_seqlens_q"),
    (dict(layout=_lib.FMLM_BWD_PADDED, seq_len=10, causal_query_seq_attn=1), "packed layout"),
    (dict(context_entries=3), "context_entries"), (dict(context_entries=1, total_context_len=5), "a context needs"),
    (dict(error_word=None), "error_word"), (dict(total_q_len=11), "view"), (dict(dq=None, dk=None, dv=None), "give dq"),
    (dict(dk=None), "give dq"), (dict(dq=(1 << 20) + 8), "aligned"), (dict(out=None), "required"),
    (dict(lse=None), "required"), (dict(workspace=None), "workspace"), (dict(workspace_bytes=256), "workspace"),
    (dict(dout=_lib.View4(1 << 20, 10, 4, 1, 128, 1280, 5120)), "contiguous"),
    (dict(dout=_lib.View4(None, 10, 4, 1, 64, 640, 2560)), "dout is required"),
])
def test_c_refusals(change, message):
    L = _lib.lib()
    assert L.fmlm_attn_bwd(ctypes.byref(bwd_args(**change)), None) == -1
    assert message in L.fmlm_last_error().decode()


def test_c_refuses_head_dim_and_null():
    L = _lib.lib()
    assert L.fmlm_attn_bwd(None, None) == -1
    assert L.fmlm_attn_dense_fwd_lse(None, 1, None, None) == -1
    assert L.fmlm_attn_packed_fwd_lse(ctypes.byref(_lib.PackedArgs()), 0, None, None) == -1
    a = bwd_args(head_dim=48)
    for f in ("q", "k", "v", "dout"):
        v = getattr(a, f)
        v.row_stride, v.head_stride = 48, 480
        setattr(a, f, v)
    assert L.fmlm_attn_bwd(ctypes.byref(a), None) == -2


@pytest.mark.parametrize("entry", ["fwd", "bwd", "train"])
@pytest.mark.parametrize("dtype,scale", [(F16, 0.0), (F16, 2.0**-25), (F16, -(2.0**21)), (F16, float("nan")),
                                         (torch.bfloat16, float("inf")), (torch.bfloat16, 2.0**65)])
def test_scale_refusals(entry, dtype, scale):
    x = z(2, 4, 8, 64, dtype=dtype)
    kw = dict(q=x, k=x, v=x, scale=scale)
    if entry == "bwd":
        kw.update(dout=x, out=x, lse=torch.zeros(2, 4, 8))
    with pytest.raises(ValueError, match="scale"):
        getattr(flash_mlm, f"flash_attn_mlm_{entry}")(**kw)


@pytest.mark.parametrize("dtype,scale", [(0, 0.0), (0, 2.0**21), (1, float("nan")), (1, 2.0**65)])
def test_c_scale_refusals(dtype, scale):
    L = _lib.lib()
    assert L.fmlm_attn_bwd(ctypes.byref(bwd_args(dtype=dtype, scale=scale)), None) == -1
    assert "scale" in L.fmlm_last_error().decode()
