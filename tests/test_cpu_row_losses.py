"""Row losses without a GPU: the header and its binding agree, every refusal comes before any device work, the oracle's gradients
are the differences of its values."""
import ctypes as C
import os
import re

import numpy as np
import pytest
import torch

from oracle import row_losses as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_header_and_binding_agree(tmp_path):
    import subprocess

    import __graft_entry__ as ge

    ge.build()
    from proximalalgorithms.jl_amd import _lib

    text = open(os.path.join(ROOT, "include", "proxgrad_hip_rows.h")).read()
    declared = set(re.findall(r"^\s*(?:pg_status|int32_t)\s+(pg_[a-z0-9_]+)\s*\(", text, flags=re.M))
    assert declared == set(_lib.exported_row_symbols())
    lib = _lib.load()
    assert all(hasattr(lib, s) for s in declared)
    assert lib.pg_rows_abi_version() == _lib.PG_ROWS_ABI_VERSION == int(re.search(r"#define PG_ROWS_ABI_VERSION (\d+)", text).group(1))
    structs = [("pg_distill", _lib.pg_distill), ("pg_balance_tile", _lib.pg_balance_tile), ("pg_balance", _lib.pg_balance)]
    src = ['#include <stdio.h>', '#include <stddef.h>', '#include "proxgrad_hip_rows.h"', "int main(void) {"]
    for name, s in structs:
        src.append(f'printf("%zu\\n", sizeof({name}));')
        src += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in s._fields_]
    (tmp_path / "a.c").write_text("\n".join(src + ["return 0; }"]))
    subprocess.run(["gcc", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(tmp_path / "a.c"), "-o", str(tmp_path / "a")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for _, s in structs:
        want += [C.sizeof(s)] + [getattr(s, f[0]).offset for f in s._fields_]
    assert got == want


def test_distillation_refusals():
    import proximalalgorithms.jl_amd as pa

    t, i = np.zeros((3, 2), np.float32), np.zeros((3, 2), np.int64)
    bad = [
        (ValueError, (t[0], i, 5), {}), (ValueError, (t, i[:2], 5), {}), (ValueError, (t, i + 5, 5), {}), (ValueError, (t, i - 2, 5), {}),
        (ValueError, (t, i, -1), {}), (ValueError, (t, i, (1 << 24) + 1), {}), (TypeError, (t, t, 5), {}), (TypeError, (i, i, 5), {}),
        (ValueError, (np.zeros((1, 1025), np.float32), np.zeros((1, 1025), int), 2000), {}),
        (ValueError, (t, i, 5), dict(temperature=0.0)), (ValueError, (t, i, 5), dict(temperature=float("inf"))),
        (ValueError, (t, i, 5), dict(lam=-1.0)), (ValueError, (t, i, 5), dict(lam=float("nan"))), (ValueError, (t, i, 5), dict(label_lam=1.0)),
        (ValueError, (t, i, 5), dict(labels=np.array([0, 5, 0]), label_lam=1.0)), (ValueError, (t, i, 5), dict(labels=np.array([0, 1]))),
        (ValueError, (t, i, 5), dict(weights=np.array([1.0, -1.0, 0.0]))), (ValueError, (t, i, 5), dict(weights=np.ones(4))),
        (ValueError, (t, i, 5), dict(teacher_lse=np.ones(2))), (TypeError, (t, i, 5), dict(teacher_lse=np.ones(3, int))),
        (TypeError, (t, i, 5), dict(labels=np.ones(3))),
    ]
    for err, args, kw in bad:
        with pytest.raises(err):
            pa.DistillationLoss(*args, **kw)
    if not torch.cuda.is_available():
        with pytest.raises(pa.ProxGradError):
            pa.DistillationLoss(t, i, 5)  # valid: and then there is no device, and no fallback


def test_balance_refusals():
    import proximalalgorithms.jl_amd as pa

    bad = [
        (ValueError, (-1, 4, 2), {}), (ValueError, (5, 0, 1), {}), (ValueError, (5, 1025, 2), {}), (ValueError, (5, 4, 0), {}), (ValueError, (5, 4, 5), {}),
        (ValueError, (5, 4, 2), dict(lam=-1.0)), (ValueError, (5, 4, 2), dict(lam=float("inf"))), (ValueError, (1 << 31, 4, 2), {}),
        (ValueError, (5, 4, 2), dict(offsets=[])), (ValueError, (5, 4, 2), dict(offsets=[1, 5])), (ValueError, (5, 4, 2), dict(offsets=[0, 3, 2])),
        (ValueError, (5, 4, 2), dict(offsets=[0, 6])), (ValueError, (5, 4, 2), dict(mask=np.ones(4, bool))), (TypeError, (5, 4, 2), dict(mask=np.ones(5))),
        (ValueError, (5, 4, 2), dict(chosen=np.zeros((5, 3), int))), (ValueError, (5, 4, 2), dict(chosen=np.full((5, 2), 4))),
        (ValueError, (5, 4, 2), dict(chosen=np.full((5, 2), -2))), (TypeError, (5, 4, 2), dict(chosen=np.zeros((5, 2)))),
        (TypeError, (5, 4, 2), dict(offsets=[0.0, 5.0])),
    ]
    for err, args, kw in bad:
        with pytest.raises(err):
            pa.BalanceLoss(*args, **kw)
    if not torch.cuda.is_available():
        with pytest.raises(pa.ProxGradError):
            pa.BalanceLoss(5, 4, 2)


def test_balance_tiles_cover_every_token_once():
    from proximalalgorithms.jl_amd.row_losses import _balance_tiles

    for tokens, offsets in ((0, [0, 0]), (1, [0, 1]), (5, [0, 0, 0, 4]), (1000, [0, 1, 1, 700, 999]), (100000, [0, 100000]), (4096, list(range(4097)))):
        tiles, size, whole = _balance_tiles(tokens, 60, offsets, 256)
        seen = np.zeros(tokens, int)
        first = set()
        for b, e, g, part in tiles:
            assert 0 <= b < e <= tokens and -1 <= g < len(offsets) - 1 and e - b <= max(size, 16)
            seen[b:e] += 1
            if g >= 0:
                assert offsets[g] <= b and e <= offsets[g + 1]
                if part <= 0:
                    assert g not in first
                    first.add(g)
                assert (part == -1) == (b == offsets[g] and e == offsets[g + 1])
        assert (seen == 1).all()
        assert first == {g for g in range(len(offsets) - 1) if offsets[g] < offsets[g + 1]}
        assert not whole or all(part == -1 or g < 0 for _, _, g, part in tiles)


def test_c_entry_refuses_before_any_device_work():
    from proximalalgorithms.jl_amd import _lib

    lib = _lib.load()
    assert lib.pg_distill_value_and_gradient(None, None, 0, None, 0, None, 0, None, None) == _lib.PG_ERR_INVALID
    assert b"null" in lib.pg_last_error()
    assert lib.pg_balance_value_and_gradient(None, None, 0, None, 0, None, 0, None, None) == _lib.PG_ERR_INVALID


@pytest.mark.parametrize("rest", [False, True])
def test_oracle_distillation_gradient_is_its_differences(rest):
    rng = np.random.default_rng(3)
    n, v, k = 3, 11, 4
    x = rng.normal(size=(n, v))
    t, idx = rng.normal(size=(n, k)) + 2, np.stack([rng.permutation(v)[:k] for _ in range(n)])
    idx[0, 3] = -1
    idx[1, 2] = idx[1, 0]
    kw = dict(temperature=1.7, lam=0.8, weights=np.array([1.0, 0.5, 2.0]), labels=np.array([-1, 2, idx[2, 0]]), label_lam=0.4)
    if rest:
        kw["teacher_lse"] = np.log(np.exp(t / 1.7).sum(1)) + 0.4
    g = ref.distillation(x, t, idx, **kw)[1]
    h = 1e-5
    for i in range(n):
        for j in range(v):
            xp, xm = x.copy(), x.copy()
            xp[i, j] += h
            xm[i, j] -= h
            d = (ref.distillation(xp, t, idx, **kw)[0] - ref.distillation(xm, t, idx, **kw)[0]) / (2 * h)
            assert abs(d - g[i, j]) < 1e-8  # second-order difference: h^2 times a third derivative of order one, plus eps / h


def test_oracle_balance_gradient_is_its_differences():
    rng = np.random.default_rng(4)
    r = rng.normal(size=(9, 6))
    kw = dict(offsets=[0, 4, 4, 8], mask=np.array([1, 1, 0, 1, 1, 1, 1, 1, 1], bool), lam=1.3)
    f, g, counts, _, _ = ref.balance(r, 2, **kw)
    assert counts.sum() == 2 * 7 and counts[1].sum() == 0 and not g[8].any() and not g[2].any()
    h = 1e-5
    for i in range(9):
        for j in range(6):
            rp, rm = r.copy(), r.copy()
            rp[i, j] += h
            rm[i, j] -= h
            fp, fm = ref.balance(rp, 2, **kw), ref.balance(rm, 2, **kw)
            assert np.array_equal(fp[2], counts) and np.array_equal(fm[2], counts)  # no choice changes within h
            assert abs((fp[0] - fm[0]) / (2 * h) - g[i, j]) < 1e-8


def test_entry_points_refuse_bad_plans_before_any_device_work():
    """every check of the C entry points that needs no device; the context is a block of zeros that none of them may look into"""
    from proximalalgorithms.jl_amd import _lib

    lib = _lib.load()
    ctx, mem = C.create_string_buffer(1 << 16), C.create_string_buffer(4096)
    base, p = C.addressof(mem), C.cast(ctx, C.c_void_p)
    good = dict(rows=2, classes=8, top=2, teacher=base, teacher_ld=2, index=base, index_ld=2, index_bits=32, temperature=1.0, lam=1.0)
    for change, dtype, ld, shift in ((dict(rows=-1), 0, 8, 0), (dict(top=1025), 0, 8, 0), (dict(classes=(1 << 24) + 1), 0, 8, 0), (dict(temperature=0.0), 0, 8, 0),
                                     (dict(temperature=float("nan")), 0, 8, 0), (dict(lam=-1.0), 0, 8, 0), (dict(label_lam=float("inf")), 0, 8, 0), (dict(teacher=None), 0, 8, 0),
                                     (dict(teacher_dtype=7), 0, 8, 0), (dict(index_bits=16), 0, 8, 0), (dict(teacher_lse=base, lse_dtype=2), 0, 8, 0),
                                     (dict(weights=base, weights_dtype=3), 0, 8, 0), (dict(labels=base, label_bits=8), 0, 8, 0), ({}, 4, 8, 0), ({}, 0, 7, 0), ({}, 0, 8, 2)):
        d = _lib.pg_distill(**{**good, **change})
        assert lib.pg_distill_value_and_gradient(p, C.byref(d), dtype, base + 64 + shift, ld, base + 2048, ld, None, None) == _lib.PG_ERR_INVALID, change
    good = dict(tokens=2, groups=1, ntiles=1, tile_tokens=2, counts=base, state=base, experts=8, k=2, copies=1, lam=1.0)
    for change, dtype, ld, shift in ((dict(tokens=-1), 0, 8, 0), (dict(tokens=1 << 31), 0, 8, 0), (dict(experts=0), 0, 8, 0), (dict(experts=1025), 0, 8, 0), (dict(k=9), 0, 8, 0),
                                     (dict(k=0), 0, 8, 0), (dict(lam=float("nan")), 0, 8, 0), (dict(ntiles=2), 0, 8, 0), (dict(groups=2), 0, 8, 0), (dict(state=None), 0, 8, 0),
                                     (dict(copies=0), 0, 8, 0), (dict(copies=17), 0, 8, 0), (dict(chosen=base, chosen_bits=16), 0, 8, 0), ({}, -1, 8, 0), ({}, 0, 7, 0), ({}, 0, 8, 1)):
        b = _lib.pg_balance(**{**good, **change})
        assert lib.pg_balance_value_and_gradient(p, C.byref(b), dtype, base + 64 + shift, ld, base + 2048, ld, None, None) == _lib.PG_ERR_INVALID, change


def test_sum_of_smooth_terms_checks_its_ranges():
    import proximalalgorithms.jl_amd as pa

    x = pa.HIPVector(None, 1024, 100, np.float32)
    for ranges in (((0, 60), (48, 100)), ((0, 101),), ((-4, 8),), ((16, 8),), ((0, 20), (0, 20))):
        with pytest.raises(ValueError):
            pa.SlicedSeparableSum((pa.SqrNormL2(),) * len(ranges), ranges).value_and_gradient(x)
    assert pa.SlicedSeparableSum((pa.SqrNormL2(), pa.Zero()), ((0, 1), (4, 8))).is_convex
    assert not pa.SlicedSeparableSum((pa.SqrNormL2(), object()), ((0, 1), (4, 8))).is_convex
