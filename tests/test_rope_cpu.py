"""CPU tests of qk_norm_rope: the C structure's layout, the table and every refusal."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import flash_mlm
from flash_mlm import _lib
from test_train_cpu import meta, z

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("gcc") is None and shutil.which("cc") is None, reason="no C compiler")
def test_args_match_header(tmp_path):
    cls, cname = _lib.QkRopeArgs, "fmlm_qk_rope_args"
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


def table(**kw):
    return flash_mlm.RotaryTable(kw.pop("n", 16), kw.pop("dim", 64), device="cpu", **kw)


def test_table_holds_float64_angles():
    t = table(n=100001, dim=16, base=10000.0).table
    assert t.shape == (100001, 8, 2) and t.dtype == torch.float32
    angle = torch.tensor(100000.0, dtype=torch.float64) * 10000.0 ** (-torch.arange(0, 16, 2, dtype=torch.float64) / 16)
    # rounded once to float32 (2^-24 of values up to 1) from float64 angles (1e5 * 2^-52 off)
    assert (t[-1, :, 0].double() - angle.cos()).abs().max() <= 2.0 ** -24 + 1e-10
    assert (t[-1, :, 1].double() - angle.sin()).abs().max() <= 2.0 ** -24 + 1e-10
    own = table(dim=16, inv_freq=torch.full((8,), 0.5))
    angle = torch.tensor(1.5, dtype=torch.float64)
    assert torch.equal(own.table[3, 0], torch.stack([angle.cos(), angle.sin()]).float())


@pytest.mark.parametrize("kw", [dict(n=0), dict(dim=24), dict(dim=0), dict(pairs="other"),
                                dict(inv_freq=torch.zeros(3))])
def test_table_refusals(kw):
    with pytest.raises(ValueError):
        table(**kw)


i32 = dict(dtype=torch.int32)
REFUSED = [
    ("rank", dict(q=z(4, 64)), "rank-4"),
    ("lengths differ", dict(k=z(2, 4, 9, 64)), "heads only"),
    ("no heads", dict(k=z(2, 0, 8, 64)), "at least one head"),
    ("head_dim", dict(q=z(2, 4, 8, 48), k=z(2, 4, 8, 48)), "HEAD_DIM"),
    ("dtype", dict(q=z(2, 4, 8, 64, dtype=torch.float32), k=z(2, 4, 8, 64, dtype=torch.float32)), "dtype"),
    ("dtypes differ", dict(k=z(2, 4, 8, 64, dtype=torch.bfloat16)), "same dtype"),
    ("packed without meta", dict(q=z(4, 8, 64), k=z(4, 8, 64)), "q_meta"),
    ("packed count", dict(q=z(4, 8, 64), k=z(4, 8, 64), q_meta=meta([3, 4], 8)), "token count"),
    ("padded meta", dict(q_meta=meta([3, 4], 9)), "padded shape"),
    ("nothing", dict(rotary=None, normalize=False), "nothing to do"),
    ("rotary_dim", dict(q=z(2, 4, 8, 32), k=z(2, 4, 8, 32)), "rotary_dim"),
    ("weights without norm", dict(normalize=False, q_weight=torch.ones(64)), "normalize"),
    ("weight shape", dict(q_weight=torch.ones(32)), r"\[head_dim\]"),
    ("weight types", dict(q_weight=torch.ones(64), k_weight=torch.ones(64, dtype=torch.float16)), "both"),
    ("weight type", dict(q_weight=torch.ones(64, dtype=torch.float64)), "both"),
    ("eps", dict(eps=-1.0), "eps"),
    ("eps nan", dict(eps=float("nan")), "eps"),
    ("positions without rotary", dict(rotary=None, positions=torch.zeros(2, 8, **i32)), "need rotary"),
    ("both", dict(positions=torch.zeros(2, 8, **i32), position_offsets=torch.zeros(2, **i32)), "not both"),
    ("positions type", dict(positions=torch.zeros(2, 8, dtype=torch.int64)), "int32"),
    ("positions shape", dict(positions=torch.zeros(16, **i32)), "int32"),
    ("offsets shape", dict(position_offsets=torch.zeros(3, **i32)), "int32"),
    ("cpu", dict(), "CUDA"),
]


@pytest.mark.parametrize("what,change,message", REFUSED, ids=[r[0] for r in REFUSED])
def test_refusals(what, change, message):
    kw = dict(q=z(2, 4, 8, 64), k=z(2, 4, 8, 64), rotary=table())
    kw.update(change)
    with pytest.raises(ValueError, match=message):
        flash_mlm.qk_norm_rope(kw.pop("q"), kw.pop("k"), kw.pop("rotary"), **kw)


def args(**change):
    """A well-formed dense argument block over made-up addresses (never launched: each test breaks one field)."""
    a = _lib.QkRopeArgs()
    a.dtype, a.head_dim, a.batch, a.seq_len, a.q_heads, a.k_heads, a.normalize = 1, 64, 2, 8, 4, 2, 1
    a.rotary_dim, a.max_positions = 64, 8
    for f, h in (("q", 4), ("k", 2), ("gq", 4), ("gk", 2)):
        setattr(a, f, _lib.View4(1 << 20, 8, h, 2, 64, 512, 512 * h))
    for f in ("table", "q_out", "k_out", "error_word", "dq_weight", "dk_weight", "workspace"):
        setattr(a, f, 1 << 20)
    a.workspace_bytes = 1 << 24
    for f, x in change.items():
        setattr(a, f, x)
    return a


@pytest.mark.parametrize("change,message", [
    (dict(dtype=5), "dtype"), (dict(batch=0), "batch"), (dict(rotary_dim=72), "rotary_dim"), (dict(rotary_dim=8), "rotary_dim"),
    (dict(pairs=2), "pairs"), (dict(table=None), "table"), (dict(max_positions=0), "table"),
    (dict(positions=1 << 20, position_offsets=1 << 20), "positions"), (dict(packed=1), "token_indices"),
    (dict(normalize=0), "weights"), (dict(error_word=None), "error_word"), (dict(q_out=None), "q_out"),
    (dict(q=_lib.View4(8, 8, 4, 2, 64, 512, 2048)), "q must be"), (dict(gk=_lib.View4(1 << 20, 8, 2, 2, 65, 512, 1024)), "gk"),
    (dict(packed=1, token_indices=1 << 20, k=_lib.View4(1 << 20, 7, 2, 1, 64, 512, 0)), "same number"),
    (dict(workspace=None), "workspace"), (dict(workspace_bytes=16), "workspace"),
])
def test_c_refusals(change, message):
    L = _lib.lib()
    assert L.fmlm_qk_rope_bwd(ctypes.byref(args(**change)), None) == -1
    assert message in L.fmlm_last_error().decode()
    assert L.fmlm_qk_rope_bwd(ctypes.byref(args(head_dim=80)), None) == -2
    assert L.fmlm_qk_rope_fwd(None, None) == -1
