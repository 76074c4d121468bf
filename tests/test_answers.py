"""dosma_amd.models.answers without a GPU: layout of the argument structs, refusals (they come before any HIP call), the
row geometry, and the 64-bit oracle against differences."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from dosma_amd import _lib as L
from dosma_amd.models import answers as A
from oracle import answers_oracle as ao

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from dosma_amd import build as hip_build

    hip_build.build()
    return L.load()


def test_struct_layout_matches_the_c_compiler(tmp_path):
    fields = {"qmri_logits": L.QmriLogits, "qmri_label_scores_args": L.QmriLabelScoresArgs, "qmri_distill_args": L.QmriDistillArgs,
              "qmri_unet2d_score_args": L.QmriUnet2dScoreArgs}
    lines, want = [], []
    for name, cls in fields.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(ctypes.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {f}));')
            want.append(getattr(cls, f).offset)
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "qmri.h"\nint main(void){\n' + "\n".join(lines) + "\nreturn 0;}\n")
    exe = tmp_path / "layout"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)])
    assert [int(v) for v in subprocess.check_output([str(exe)]).decode().split()] == want
    head = open(os.path.join(ROOT, "include", "qmri.h")).read()
    assert f"#define QMRI_MAX_TOP {L.MAX_TOP} " in head and f"#define QMRI_SHORT_ROW {L.SHORT_ROW} " in head


def _scores_args(**kw):
    buf = np.zeros(64, np.float32)
    a = L.QmriLabelScoresArgs()
    L._fill_logits(a, buf.ctypes.data, "float32", L.Rows(2, 4), 1.0, False)
    a.entropy = a.norm = a.grad = buf.ctypes.data
    a.grad_stride_inner, a.grad_stride_class = 4, 1
    for k, v in kw.items():
        if k in ("dtype", "rows", "inner", "classes", "background", "stride_inner", "stride_class", "temperature", "data"):
            setattr(a.logits, k, v)
        else:
            setattr(a, k, v)
    a._keep = buf
    return a


def _distill_args(**kw):
    buf = np.zeros(64, np.float32)
    a = L.QmriDistillArgs()
    L._fill_logits(a, buf.ctypes.data, "float32", L.Rows(2, 4), 1.0, False)
    a.top_label = a.values = a.norm = a.grad_loss = a.grad = buf.ctypes.data
    a.entries, a.grad_stride_inner, a.grad_stride_class = 2, 4, 1
    for k, v in kw.items():
        setattr(a.logits if hasattr(a.logits, k) and k not in ("reserved",) else a, k, v)
    a._keep = buf
    return a


@pytest.mark.parametrize("bad, says", [
    (dict(dtype=1), b"logits must be"), (dict(dtype=9), b"logits must be"), (dict(rows=-1), b"rows"), (dict(classes=0), b"classes"),
    (dict(background=2), b"background"), (dict(inner=0), b"inner"), (dict(stride_class=-1), b"negative stride"),
    (dict(temperature=0.0), b"temperature"), (dict(temperature=-1.0), b"temperature"), (dict(temperature=float("nan")), b"temperature"),
    (dict(temperature=float("inf")), b"temperature"), (dict(device=-1), b"device"), (dict(device=99), b"device"), (dict(data=None), b"NULL"),
    (dict(top=-1), b"top"), (dict(top=65), b"top"), (dict(top=5), b"categories"), (dict(top=2), b"top_log_prob"),
    (dict(log_prob=16), b"needs labels"), (dict(labels=16, l_kind=7), b"l_kind"),
])
def test_label_scores_refusals(lib, bad, says):
    for entry in (lib.qmri_label_scores_device, lib.qmri_label_scores_host):
        assert entry(ctypes.byref(_scores_args(**bad))) == L.QMRI_ERR_ARG
        assert says in lib.qmri_last_error()


@pytest.mark.parametrize("bad, says", [
    (dict(grad=None), b"grad is NULL"), (dict(norm=None), b"norm"), (dict(grad_log_prob=16), b"needs labels"),
    (dict(grad_entropy=16, entropy=None), b"needs entropy"), (dict(grad_stride_class=0), b"place of its own"),
    (dict(grad_stride_inner=0), b"place of its own"), (dict(dtype=3), b"logits must be"),
])
def test_label_scores_grad_refusals(lib, bad, says):
    for entry in (lib.qmri_label_scores_grad_device, lib.qmri_label_scores_grad_host):
        assert entry(ctypes.byref(_scores_args(**bad))) == L.QMRI_ERR_ARG
        assert says in lib.qmri_last_error()


@pytest.mark.parametrize("bad, says", [
    (dict(entries=0), b"entries"), (dict(entries=65), b"entries"), (dict(l_kind=1), b"teacher labels"), (dict(tail=2), b"tail"),
    (dict(v_dtype=1), b"values must be"), (dict(tail=1, v_dtype=4), b"float32 log"), (dict(values=None), b"NULL"),
    (dict(top_label=None), b"NULL"), (dict(temperature=0.0), b"temperature"), (dict(classes=0), b"classes"),
])
def test_distill_refusals(lib, bad, says):
    for entry in (lib.qmri_distill_device, lib.qmri_distill_host, lib.qmri_distill_grad_device, lib.qmri_distill_grad_host):
        assert entry(ctypes.byref(_distill_args(**bad))) == L.QMRI_ERR_ARG
        assert says in lib.qmri_last_error()


def test_distill_grad_refusals(lib):
    for bad, says in ((dict(grad=None), b"grad is NULL"), (dict(norm=None), b"norm"), (dict(grad_loss=None), b"grad_loss"),
                      (dict(tail=1), b"log_tail"), (dict(grad_stride_class=0), b"place of its own")):
        assert lib.qmri_distill_grad_device(ctypes.byref(_distill_args(**bad))) == L.QMRI_ERR_ARG
        assert says in lib.qmri_last_error()


def test_null_and_empty_calls(lib):
    for name in ("label_scores", "distill"):
        for entry in ("device", "host", "grad_device", "grad_host"):
            assert getattr(lib, f"qmri_{name}_{entry}")(None) == L.QMRI_ERR_ARG
    n = ctypes.c_uint64(7)
    assert lib.qmri_label_scores_workspace(None, ctypes.byref(n)) == L.QMRI_ERR_ARG
    assert lib.qmri_label_scores_workspace(ctypes.byref(_scores_args()), None) == L.QMRI_ERR_ARG
    assert lib.qmri_label_scores_device(ctypes.byref(_scores_args(rows=0, data=None))) == L.QMRI_OK  # nothing to do
    assert lib.qmri_distill_device(ctypes.byref(_distill_args(rows=0, data=None))) == L.QMRI_OK


def test_host_entry_takes_dense_rows(lib):
    assert lib.qmri_label_scores_host(ctypes.byref(_scores_args(stride_inner=5))) == L.QMRI_ERR_ARG
    assert b"dense rows" in lib.qmri_last_error()
    assert lib.qmri_distill_host(ctypes.byref(_distill_args(stride_class=2))) == L.QMRI_ERR_ARG
    assert b"dense rows" in lib.qmri_last_error()


def test_python_refusals():
    import torch

    z = np.zeros((3, 4), np.float32)
    for call, says in (
            (lambda: A.label_scores(z, np.zeros(2, np.int32)), "labels has shape"),
            (lambda: A.label_scores(z, np.zeros(3, np.uint16)), "labels must be one of"),
            (lambda: A.label_scores(z, np.zeros(3, np.float32)), "labels must be one of"),
            (lambda: A.label_scores(z.astype(np.int32)), "floating point"),
            (lambda: A.label_scores(z, top=65), "top"),
            (lambda: A.label_scores(z, top=-1), "top"),
            (lambda: A.label_scores(z, dim=2), "dim"),
            (lambda: A.label_scores(np.float32(1.0)), "class axis"),
            (lambda: A.distill_loss(z, np.zeros((3, 2), np.int32), np.zeros((3, 3), np.float32)), "values has shape"),
            (lambda: A.distill_loss(z, np.zeros((2, 2), np.int32), np.zeros((2, 2), np.float32)), "top_label has shape"),
            (lambda: A.distill_loss(z, np.zeros((3, 2), np.uint8), np.zeros((3, 2), np.float32)), "top_label must be one of"),
            (lambda: A.label_scores_grad(z, None, np.zeros((3, 1), np.float32)), "norm has shape"),
            (lambda: A.distill_loss_grad(z, np.zeros((3, 2), np.int32), np.zeros((3, 2), np.float32), np.zeros((3, 2), np.float32),
                                         grad_loss=np.zeros(3)), "grad_loss must be one of"),
            (lambda: A.label_scores(torch.zeros(3, 4)), "on the GPU"),
            (lambda: A.distill_loss(torch.zeros(3, 4), torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, 1)), "on the GPU")):
        with pytest.raises(ValueError, match=says):
            call()


def test_no_cpu_fallback(lib):
    if lib.qmri_device_count() > 0:
        pytest.skip("a GPU is present")
    z = np.zeros((3, 4), np.float32)
    with pytest.raises(L.QmriError):
        A.label_scores(z)
    with pytest.raises(L.QmriError):
        A.distill_loss(z, np.zeros((3, 2), np.int32), np.zeros((3, 2), np.float32))


@pytest.mark.parametrize("shape, strides, dim, want", [
    ((6, 4), (4, 1), 1, (6, 4, 6, 0, 4, 1)), ((6, 4), (9, 1), 1, (6, 4, 6, 0, 9, 1)), ((2, 4, 3, 5), (60, 15, 5, 1), 1, (30, 4, 15, 60, 1, 15)),
    ((2, 3, 5, 4), (60, 20, 4, 1), 3, (30, 4, 30, 0, 4, 1)), ((4,), (1,), 0, (1, 4, 1, 0, 4, 1)), ((1, 4), (100, 1), 1, (1, 4, 1, 0, 4, 1)),
    ((7, 4), (0, 1), 1, (7, 4, 7, 0, 0, 1)), ((7, 4), (4, 0), 1, (7, 4, 7, 0, 4, 0)), ((4, 7), (7, 1), 0, (7, 4, 7, 0, 1, 7)),
    ((3, 1, 5), (5, 5, 1), 1, (15, 1, 15, 0, 1, 1)), ((0, 4), (4, 1), 1, (0, 4, 1, 0, 4, 1)),
    ((2, 3, 5, 4), (1000, 100, 7, 1), 3, None), ((2, 3, 4), (12, 4, 1), 2, (6, 4, 6, 0, 4, 1)), ((2, 3, 4), (4, 8, 1), 2, (6, 4, 3, 4, 8, 1)),
])
def test_row_geometry(shape, strides, dim, want):
    row_shape, r = A._rows_of(shape, strides, dim)
    assert row_shape == shape[:dim] + shape[dim + 1:]
    if want is None:
        assert r is None
        return
    assert (r.rows, r.classes, r.inner, r.so, r.si, r.sc) == want
    # the element every (row, class) addresses is numpy's
    at = 0
    for idx in np.ndindex(*row_shape):
        full = list(idx)
        full.insert(dim, 0)
        n = int(np.ravel_multi_index(idx, row_shape)) if row_shape else 0
        at = sum(i * s for i, s in zip(full, strides))
        assert at == (n // r.inner) * r.so + (n % r.inner) * r.si


def test_oracle_gradients_against_differences():
    """The 64-bit definitions the GPU is held to: central differences with h = 1e-5 are off by h^2 f''' / 6 ~ 1e-11 and the
    rounding 1e-16 / h ~ 1e-11 of O(1) sums: 1e-8 leaves a factor of 100."""
    rng = np.random.default_rng(0)
    z = rng.standard_normal((5, 6)) * 2
    lab = np.array([0, 5, -1, 2, 3])
    a, b, w = rng.standard_normal(5), rng.standard_normal(5), rng.standard_normal(5)
    ti = np.array([[0, 1], [5, 5], [-1, 3], [-1, -1], [2, 4]])
    tv = np.log(rng.uniform(0.1, 0.4, (5, 2)))
    for T in (0.7, 2.0):
        f = lambda x: np.sum(a * ao.scores(x, T, lab)["log_prob"] + b * ao.scores(x, T)["entropy"])  # noqa: E731
        fs = [(f, ao.scores_grad(z, T, lab, a, b))]
        for tail in (False, True):
            fs.append((lambda x, t=tail: np.sum(w * ao.distill(x, ti, tv, T, t)["loss"]), ao.distill(z, ti, tv, T, tail, w)["grad"]))
        for fn, g in fs:
            num = np.zeros_like(z)
            for i in np.ndindex(*z.shape):
                up, dn = z.copy(), z.copy()
                up[i] += 1e-5
                dn[i] -= 1e-5
                num[i] = (fn(up) - fn(dn)) / 2e-5
            assert np.abs(num - g).max() < 1e-8


def test_gradients_rows_that_meet_are_refused(lib):
    """The row axis and the class axis of a gradient must not share places: one group of 6 rows a step apart, classes 3 apart."""
    for bad in (dict(rows=6, inner=6, grad_stride_inner=1, grad_stride_class=3), dict(grad_stride_inner=2, grad_stride_class=2),
                dict(rows=6, inner=3, grad_stride_inner=4, grad_stride_outer=8), dict(rows=6, inner=3, grad_stride_inner=9, grad_stride_outer=3)):
        assert lib.qmri_label_scores_grad_device(ctypes.byref(_scores_args(**bad))) == L.QMRI_ERR_ARG
        assert b"place of its own" in lib.qmri_last_error()
        assert lib.qmri_distill_grad_device(ctypes.byref(_distill_args(**bad))) == L.QMRI_ERR_ARG
        assert b"place of its own" in lib.qmri_last_error()


def random_layout(rng, shape, make):
    """A view of ``shape`` of what ``make(shape)`` gives: permuted in memory, cropped, in steps, repeated."""
    nd = len(shape)
    order = rng.permutation(nd) if rng.random() < 0.6 else np.arange(nd)
    big, cut, rep = [], [], []
    for n in shape:
        kind = rng.choice(["whole", "whole", "crop", "step", "repeat"])
        first, step = (int(rng.integers(0, 3)), 1) if kind == "crop" else (int(rng.integers(0, 2)), int(rng.integers(2, 4))) if kind == "step" else (0, 1)
        big.append(1 if kind == "repeat" else first + step * n + (int(rng.integers(0, 2)) if kind == "crop" else 0))
        cut.append(slice(first, first + step * n, step))
        rep.append(kind == "repeat")
    t = make([big[i] for i in order]).permute(*[int(i) for i in np.argsort(order)])
    t = t[tuple(slice(None) if r else c for c, r in zip(cut, rep))]
    t = t[tuple(slice(0, n) for n in shape)]
    return t.expand(*shape)


def _addresses(shape, strides, dim):
    """(rows, classes) offsets of the elements."""
    at = np.zeros(shape, np.int64)
    for i, (n, st) in enumerate(zip(shape, strides)):
        at += (np.arange(n) * st).reshape([-1 if k == i else 1 for k in range(len(shape))])
    return np.moveaxis(at, dim, -1).reshape(-1, shape[dim])


def test_scores_and_gradient_are_walked_through_together():
    """The kernels count the rows of both by one ``inner``: over random crops, steps, repeats and orders of the axes every score's
    and every gradient's element is numpy's, and the gradient has a place for each."""
    import torch

    call = object.__new__(A._TorchCall)  # (its constructor asks for a stream)
    call.torch = torch
    rng = np.random.default_rng(12)
    seen = set()
    for turn in range(4000):
        nd = int(rng.integers(1, 5))
        shape = tuple(int(v) for v in rng.integers(1, 5, nd))
        x = random_layout(rng, shape, lambda s: torch.zeros(s))
        assert tuple(x.shape) == shape
        dim = int(rng.integers(0, nd))
        y, (_, rows) = x, A._rows_of(shape, x.stride(), dim)
        if rows is None:  # as _tensor_logits
            y = x.contiguous()
            rows = A._rows_of(shape, y.stride(), dim)[1]
        z, rows, g, grad_rows = call.grad_like(y, dim, rows)
        assert g.shape == x.shape and g.dtype == x.dtype and rows.rows == grad_rows.rows and rows.classes == shape[dim]
        n = np.arange(rows.rows)[:, None]
        j = np.arange(rows.classes)[None]
        for t, r in ((z, rows), (g, grad_rows)):
            got = (n // rows.inner) * r.so + (n % rows.inner) * r.si + j * r.sc
            assert np.array_equal(got, _addresses(shape, t.stride(), dim)), (shape, x.stride(), g.stride(), dim)
        assert len(np.unique(_addresses(shape, g.stride(), dim))) == g.numel()
        a = L.QmriLabelScoresArgs()
        L._fill_logits(a, 0, "float32", rows, 1.0, False)
        L._fill_grad(a, 0, grad_rows)  # (refuses rows counted differently)
        seen.add((z is x, rows.inner == rows.rows, g.is_contiguous()))
    assert len(seen) >= 6
    a = L.QmriLabelScoresArgs()
    L._fill_logits(a, 0, "float32", L.Rows(6, 4, 3, 100, 4, 1), 1.0, False)
    with pytest.raises(ValueError, match="counted by"):
        L._fill_grad(a, 0, L.Rows(6, 4))


@pytest.mark.parametrize("shape, make, dim", [
    ((2, 5, 7), lambda t: t[:, :-1], -1), ((2, 5, 7), lambda t: t[:, 1:], -1), ((2, 6, 5, 4), lambda t: t.permute(0, 3, 1, 2)[:, :, 1:-1, 2:], 1),
    ((2, 6, 5, 4), lambda t: t.permute(0, 3, 1, 2)[:, :, :, 2:], 1), ((9, 8, 3, 4), lambda t: t[2:-2, 1:-1], -1), ((1, 4, 1), lambda t: t.expand(3, 4, 5), 1), ((3, 1, 6), lambda t: t.expand(3, 5, 6), 2),
])
def test_layouts_that_a_gradient_is_asked_for(shape, make, dim):
    import torch

    call = object.__new__(A._TorchCall)
    call.torch = torch
    x = make(torch.zeros(shape))
    d = dim % x.ndim
    rows = A._rows_of(x.shape, x.stride(), d)[1]
    if rows is None:  # (cropped in H and in W of (B, H, W): three strides, copied before)
        assert shape == (2, 6, 5, 4) and x.shape[2] == 4
        x = x.contiguous()
        rows = A._rows_of(x.shape, x.stride(), d)[1]
    z, rows, g, grad_rows = call.grad_like(x, d, rows)
    assert z is x  # no copy
    n, j = np.arange(rows.rows)[:, None], np.arange(rows.classes)[None]
    for t, r in ((x, rows), (g, grad_rows)):
        assert np.array_equal((n // rows.inner) * r.so + (n % rows.inner) * r.si + j * r.sc, _addresses(tuple(x.shape), t.stride(), d))


def test_a_single_rows_arguments_have_no_axis():
    for label in (2, np.int32(2), np.array(2, np.uint8)):
        a = A._array_arg("labels", label, (), L.L_KINDS)
        assert a.shape == () and a == 2
    assert A._array_arg("norm", np.zeros(2, np.float32), (), ("float32",), 2).shape == (2,)
    with pytest.raises(ValueError, match="labels has shape"):
        A._array_arg("labels", np.zeros(1, np.int32), (), L.L_KINDS)
    t = np.arange(6, dtype=np.int32).reshape(2, 3).T
    assert A._array_arg("labels", t, (3, 2), L.L_KINDS).flags.c_contiguous


def test_arrays_of_the_other_byte_order():
    """As files hold them (big-endian label volumes): the type's name is the same, the bytes are not."""
    lab = np.array([0, 1, 2], np.int32)
    for t in (">i4", ">i2", ">i8", "<i4", "u1"):
        a = A._array_arg("labels", lab.astype(t), (3,), L.L_KINDS)
        assert a.dtype.isnative and np.array_equal(a, lab) and np.array_equal(np.frombuffer(a.tobytes(), a.dtype.name), lab)
    for t in (">f4", ">f2", ">f8", "f8", "f4"):
        _, v, _ = A._teacher_arrays(lab[:, None], np.array([[0.5], [-2.0], [7.0]]).astype(t), (3,), False)
        assert v.dtype.isnative and v.dtype.itemsize < 8 and np.array_equal(v[:, 0], [0.5, -2.0, 7.0])
    for t in (">f4", ">f2", ">f8"):
        x, _, _, _ = A._array_logits(np.array([[0.5, -2.0]]).astype(t), -1)
        assert x.dtype.isnative and np.array_equal(x[0], [0.5, -2.0])
