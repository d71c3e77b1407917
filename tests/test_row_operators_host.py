"""Host side of dropout, the layer norm and the adapters: the packed structures are the C ones, what the calls refuse is refused
before a device is touched, and nothing runs without one."""
import ctypes as C
import struct

import pytest
import torch

from cellerator_b200 import capi, ops
from row_operators import philox_words

ADDRESS = 1 << 20                                             # never followed


def dropout(**change):
    d = capi.Dropout(probability=0.1, seed=1, sequence=2, device_sequence=None, first_row=0)
    for k, v in change.items():
        setattr(d, k, v)
    return d


def drop_matrix(**change):
    m = capi.header(capi.DropoutMatrix())
    m.rows, m.columns, m.x, m.x_ld, m.y, m.y_ld = 4, 8, ADDRESS, 8, 2 * ADDRESS, 8
    m.x_dtype = m.y_dtype = capi.DTYPE_F32
    m.dropout = dropout()
    for k, v in change.items():
        setattr(m, k, v)
    return m


def norm(**change):
    n = capi.header(capi.LayerNorm())
    n.rows, n.columns, n.x, n.x_ld, n.epsilon = 4, 8, ADDRESS, 8, 1e-5
    n.y, n.dy, n.dx = 2 * ADDRESS, 3 * ADDRESS, 4 * ADDRESS
    n.y_ld = n.dy_ld = n.dx_ld = 8
    n.x_dtype = n.y_dtype = n.dy_dtype = n.dx_dtype = capi.DTYPE_F32
    n.stats, n.dgamma, n.dbeta, n.workspace, n.workspace_bytes = 5 * ADDRESS, 6 * ADDRESS, 7 * ADDRESS, 8 * ADDRESS, 1 << 20
    for k, v in change.items():
        setattr(n, k, v)
    return n


def adapters(csr=None, **change):
    x = capi.header(capi.QCsr())
    x.rows, x.cols, x.nnz, x.bits, x.policy = 4, 16, 10, 8, 1
    x.row_ptr = x.col_idx = x.packed_values = ADDRESS
    for k, v in (csr or {}).items():
        setattr(x, k, v)
    a = capi.header(capi.Adapters())
    a.csr = C.pointer(x)
    a.adapter, a.adapters, a.rank, a.n, a.down, a.up, a.weight_dtype = ADDRESS, 2, 8, 32, ADDRESS, ADDRESS, capi.DTYPE_F32
    a.out, a.out_ld, a.alpha, a.row_end = 2 * ADDRESS, 32, 1.0, capi.ALL_ROWS
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("packer,structure", [(ops._DROPOUT_MATRIX, capi.DropoutMatrix), (ops._LAYER_NORM, capi.LayerNorm),
                                              (ops._ADAPTERS, capi.Adapters)])
def test_packed_structures_have_the_fields_where_c_has_them(packer, structure):
    def leaves(s, prefix=()):
        for name, kind in s._fields_:
            if hasattr(kind, "_fields_") and issubclass(kind, C.Structure):
                yield from leaves(kind, prefix + (name,))
            else:
                yield prefix + (name,), kind
    fields = list(leaves(structure))
    values = [float(i + 1) if kind in (C.c_float, C.c_double) else i + 1 for i, (_, kind) in enumerate(fields)]
    s = structure.from_buffer_copy(packer.pack(*values))
    for (path, kind), value in zip(fields, values):
        v = s
        for name in path:
            v = getattr(v, name)
        if not isinstance(v, (int, float)):
            v = C.cast(v, C.c_void_p).value
        assert v == value, path


def test_the_generator_of_the_tests_gives_the_published_words():
    """Known answers of Philox4x32-10 published with the generator: counter and key all zeros, and all ones."""
    assert [hex(v) for v in philox_words(1, 4, 0, 0)[0].tolist()] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]
    ones = 0xFFFFFFFF
    # column / 4 = 2^32 - 1 is no width that a test can write out: the words through one round at a time
    a = b = c = d = k0 = k1 = ones
    for _ in range(10):
        p, q = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = (q >> 32) ^ b ^ k0, q & ones, (p >> 32) ^ d ^ k1, p & ones
        k0, k1 = (k0 + 0x9E3779B9) & ones, (k1 + 0xBB67AE85) & ones
    assert [hex(v) for v in (a, b, c, d)] == ["0x408f276d", "0x41c83b0e", "0xa20bc7c6", "0x6d5451fd"]


@pytest.mark.parametrize("change,status", [
    (dict(version=1), capi.INVALID_ARGUMENT), (dict(size=8), capi.INVALID_ARGUMENT),
    (dict(rows=-1), capi.INVALID_SHAPE), (dict(columns=-1), capi.INVALID_SHAPE), (dict(rows=2 ** 32 + 1), capi.INVALID_SHAPE),
    (dict(columns=2 ** 30 + 4, x_ld=2 ** 30 + 4, y_ld=2 ** 30 + 4, rows=1), capi.INVALID_SHAPE), (dict(x_ld=7), capi.INVALID_SHAPE), (dict(y_ld=7), capi.INVALID_SHAPE),
    (dict(x_ld=2 ** 62), capi.INVALID_SHAPE), (dict(x=None), capi.INVALID_ARGUMENT), (dict(y=None), capi.INVALID_ARGUMENT),
    (dict(x=ADDRESS + 2), capi.INVALID_ARGUMENT), (dict(x_dtype=capi.DTYPE_F64), capi.UNSUPPORTED), (dict(y_dtype=capi.DTYPE_U8), capi.UNSUPPORTED),
    (dict(y=ADDRESS + 4), capi.INVALID_ARGUMENT), (dict(y=ADDRESS + 32 * 3), capi.INVALID_ARGUMENT),
    (dict(y=ADDRESS, y_dtype=capi.DTYPE_F16), capi.INVALID_ARGUMENT), (dict(y=ADDRESS, y_ld=9), capi.INVALID_ARGUMENT),
    (dict(dropout=dropout(probability=1.0)), capi.INVALID_ARGUMENT), (dict(dropout=dropout(probability=-0.1)), capi.INVALID_ARGUMENT),
    (dict(dropout=dropout(probability=float("nan"))), capi.INVALID_ARGUMENT), (dict(dropout=dropout(first_row=-1)), capi.INVALID_SHAPE),
    (dict(dropout=dropout(first_row=2 ** 32 - 3)), capi.INVALID_SHAPE), (dict(dropout=dropout(device_sequence=12)), capi.INVALID_ARGUMENT),
])
def test_dropout_refuses(change, status):
    assert capi.lib().cb200_dropout_rows(C.byref(drop_matrix(**change)), None) == status
    assert capi.lib().cb200_last_error()


@pytest.mark.parametrize("change,status", [
    (dict(version=1), capi.INVALID_ARGUMENT), (dict(rows=-1), capi.INVALID_SHAPE), (dict(columns=0), capi.INVALID_SHAPE),
    (dict(columns=65_537, x_ld=65_537), capi.INVALID_SHAPE), (dict(x_ld=7), capi.INVALID_SHAPE), (dict(x=None), capi.INVALID_ARGUMENT),
    (dict(x_dtype=capi.DTYPE_F64), capi.UNSUPPORTED), (dict(gamma=ADDRESS + 1), capi.INVALID_ARGUMENT), (dict(stats=ADDRESS + 4), capi.INVALID_ARGUMENT),
    (dict(epilogue=1), capi.UNSUPPORTED), (dict(epilogue=5), capi.UNSUPPORTED), (dict(epilogue=9), capi.UNSUPPORTED), (dict(epilogue=-1), capi.UNSUPPORTED),
    (dict(dropout=dropout(probability=1.5)), capi.INVALID_ARGUMENT),
])
def test_layer_norm_refuses_both_ways(change, status):
    assert capi.lib().cb200_layer_norm_forward(C.byref(norm(**change)), None) == status
    assert capi.lib().cb200_layer_norm_backward(C.byref(norm(**change)), None) == status
    assert capi.lib().cb200_last_error()


@pytest.mark.parametrize("change,status", [
    (dict(epsilon=-1.0), capi.INVALID_ARGUMENT), (dict(epsilon=float("nan")), capi.INVALID_ARGUMENT), (dict(epsilon=float("inf")), capi.INVALID_ARGUMENT),
    (dict(y=None), capi.INVALID_ARGUMENT), (dict(y_ld=3), capi.INVALID_SHAPE), (dict(y=ADDRESS + 16), capi.INVALID_ARGUMENT),
    (dict(y=ADDRESS, y_dtype=capi.DTYPE_BF16), capi.INVALID_ARGUMENT), (dict(y_dtype=0), capi.UNSUPPORTED),
])
def test_layer_norm_forward_refuses(change, status):
    assert capi.lib().cb200_layer_norm_forward(C.byref(norm(**change)), None) == status


@pytest.mark.parametrize("change,status", [
    (dict(dy=None), capi.INVALID_ARGUMENT), (dict(dy_ld=3), capi.INVALID_SHAPE), (dict(stats=None), capi.INVALID_ARGUMENT),
    (dict(dx=ADDRESS + 16), capi.INVALID_ARGUMENT), (dict(dx=3 * ADDRESS + 16), capi.INVALID_ARGUMENT), (dict(dx_dtype=0), capi.UNSUPPORTED),
    (dict(workspace=None), capi.INSUFFICIENT_WORKSPACE), (dict(workspace_bytes=3), capi.INSUFFICIENT_WORKSPACE),
    (dict(workspace=ADDRESS + 2), capi.INSUFFICIENT_WORKSPACE),
    (dict(columns=5000, x_ld=5000, dy_ld=5000, dx_ld=5000, dx=ADDRESS, dgamma=None, dbeta=None, workspace=None), capi.INSUFFICIENT_WORKSPACE), (dict(dgamma=ADDRESS * 9, dbeta=ADDRESS * 9), capi.INVALID_ARGUMENT),
])
def test_layer_norm_backward_refuses(change, status):
    assert capi.lib().cb200_layer_norm_backward(C.byref(norm(**change)), None) == status


def test_layer_norm_workspace():
    """Two sums per column of every part, as the header says, and a bound on the parts; of wide rows two per row and 4,096 columns."""
    assert ops.layer_norm_backward_workspace(0, 64) == 0
    assert ops.layer_norm_backward_workspace(1, 64) == 2 * 64 * 4
    assert ops.layer_norm_backward_workspace(1_000_000, 64) <= 2 * 64 * 4 * 1024
    assert ops.layer_norm_backward_workspace(1_000_000, 33_538) <= 2 * 33_538 * 4 * 128 + 1_000_000 * 9 * 8
    for bad in ((-1, 8), (8, 0), (8, 65_537)):
        with pytest.raises(capi.Cb200Error):
            ops.layer_norm_backward_workspace(*bad)
    assert capi.lib().cb200_layer_norm_backward_workspace(8, 8, None) == capi.INVALID_ARGUMENT


@pytest.mark.parametrize("change,csr,status", [
    (dict(version=1), {}, capi.INVALID_ARGUMENT), ({}, dict(version=1), capi.INVALID_ARGUMENT), ({}, dict(bits=2), capi.UNSUPPORTED),
    ({}, dict(policy=3), capi.UNSUPPORTED), ({}, dict(bits=4), capi.INVALID_ARGUMENT), (dict(weight_dtype=capi.DTYPE_F16), {}, capi.UNSUPPORTED),
    (dict(epilogue=8), {}, capi.UNSUPPORTED), (dict(epilogue=1), {}, capi.INVALID_ARGUMENT), (dict(rank=0), {}, capi.UNSUPPORTED),
    (dict(rank=257), {}, capi.UNSUPPORTED), (dict(n=-1), {}, capi.INVALID_SHAPE), (dict(adapters=-1), {}, capi.INVALID_SHAPE),
    (dict(out_ld=31), {}, capi.INVALID_SHAPE), (dict(row_begin=-1), {}, capi.INVALID_SHAPE), (dict(row_begin=3, row_end=2), {}, capi.INVALID_SHAPE),
    (dict(row_end=5), {}, capi.INVALID_SHAPE), (dict(adapter=None), {}, capi.INVALID_ARGUMENT), (dict(out=None), {}, capi.INVALID_ARGUMENT),
    (dict(down=None), {}, capi.INVALID_ARGUMENT), (dict(up=None), {}, capi.INVALID_ARGUMENT), (dict(up=ADDRESS + 2), {}, capi.INVALID_ARGUMENT),
    (dict(scale=ADDRESS + 2), {}, capi.INVALID_ARGUMENT), (dict(bias=ADDRESS + 2, epilogue=1), {}, capi.INVALID_ARGUMENT),
    ({}, dict(row_ptr=ADDRESS + 4), capi.INVALID_ARGUMENT), ({}, dict(bits=4, packed_row_ptr=ADDRESS + 4), capi.INVALID_ARGUMENT),
    ({}, dict(col_idx=ADDRESS + 2), capi.INVALID_ARGUMENT), ({}, dict(scales=ADDRESS + 1), capi.INVALID_ARGUMENT),
    ({}, dict(offsets=ADDRESS + 1), capi.INVALID_ARGUMENT),
    ({}, dict(row_ptr=None), capi.INVALID_ARGUMENT), ({}, dict(col_idx=None), capi.INVALID_ARGUMENT), ({}, dict(rows=-1), capi.INVALID_SHAPE),
])
def test_adapters_refuse(change, csr, status):
    assert capi.lib().cb200_qcsr_adapters(C.byref(adapters(csr, **change)), None) == status
    assert capi.lib().cb200_last_error()


def test_null_descriptors_are_refused():
    L = capi.lib()
    assert L.cb200_dropout_rows(None, None) == L.cb200_layer_norm_forward(None, None) == L.cb200_layer_norm_backward(None, None) \
        == L.cb200_qcsr_adapters(None, None) == capi.INVALID_ARGUMENT


@pytest.mark.parametrize("y,y_ld", [(ADDRESS, 8), (ADDRESS + 4 * 32, 8), (2 * ADDRESS, 20)])
def test_no_cpu_fallback_without_a_device(y, y_ld):
    """... and what stands beside x or is x is not refused: without a device such a call gets as far as that."""
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")
    L = capi.lib()
    assert L.cb200_dropout_rows(C.byref(drop_matrix(y=y, y_ld=y_ld)), None) == capi.CUDA_ERROR
    assert L.cb200_layer_norm_forward(C.byref(norm(y=y, y_ld=y_ld)), None) == capi.CUDA_ERROR
    assert L.cb200_layer_norm_backward(C.byref(norm(dx=y, dx_ld=y_ld)), None) == capi.CUDA_ERROR
    assert L.cb200_qcsr_adapters(C.byref(adapters()), None) == capi.CUDA_ERROR


def test_columns_side_by_side_in_one_buffer_do_not_overlap():
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is present")                 # what is not refused would run
    L = capi.lib()
    # x in columns 0..7, y in 8..15 of rows of 16; then one column further to the left, and out of the row's end into the next one
    status = [L.cb200_dropout_rows(C.byref(drop_matrix(x_ld=16, y_ld=16, y=ADDRESS + 4 * at)), None) for at in (8, 7, 9, 24, 25, -8, -7)]
    refused = [s == capi.INVALID_ARGUMENT for s in status]
    assert refused == [False, True, True, False, True, False, True]


def test_python_checks():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ops.dropout(x, 0.1, 1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.layer_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.layer_norm_backward(x, x, torch.zeros(4, 2))
    for bad in (x.double(), x[0], x.t(), x[:, ::2]):
        with pytest.raises(ValueError):
            ops.dropout(bad, 0.1, 1)
        with pytest.raises(ValueError):
            ops.layer_norm(bad)
    for bad in (dict(seed=-1), dict(seed=1 << 64), dict(seed=1, sequence=-1), dict(seed=1, device_sequence=torch.zeros(1))):
        with pytest.raises(ValueError, match="whole number"):
            ops.dropout(x, 0.1, **bad)
    for bad in (dict(gamma=torch.ones(7)), dict(gamma=torch.ones(8).double()), dict(beta=torch.ones(16)[::2]), dict(stats=torch.zeros(2, 4)),
                dict(out=torch.zeros(4, 9)), dict(out=x, out_dtype=torch.float16)):
        with pytest.raises(ValueError):
            ops.layer_norm(x, **bad)
    for bad in (dict(dy=torch.zeros(5, 8)), dict(stats=torch.zeros(4, 2).half()), dict(dx=x, dx_dtype=torch.float16), dict(dgamma=torch.zeros(9)),
                dict(workspace=torch.zeros(4096)[::2])):
        with pytest.raises(ValueError):
            ops.layer_norm_backward(x, **{**dict(dy=x, stats=torch.zeros(4, 2)), **bad})


def test_python_checks_of_adapters():
    m = ops.QuantizedCsr(3, 6, 8, 1, torch.zeros(4, dtype=torch.int64), torch.zeros(0, dtype=torch.int32), torch.zeros(0, dtype=torch.uint8), None, None)
    good = dict(adapter=torch.zeros(3, dtype=torch.int32), down=torch.zeros(2, 6, 4), up=torch.zeros(2, 4, 5))
    with pytest.raises(ValueError, match="CUDA"):
        ops.adapter_forward(m, **good)
    for bad in (dict(adapter=torch.zeros(3)), dict(adapter=torch.zeros(4, dtype=torch.int32)), dict(down=torch.zeros(2, 7, 4)), dict(up=torch.zeros(2, 3, 5)),
                dict(up=torch.zeros(1, 4, 5)), dict(up=torch.zeros(2, 4, 5).bfloat16()), dict(down=torch.zeros(2, 4, 6).transpose(1, 2)),
                dict(scale=torch.zeros(3)), dict(bias=torch.zeros(4)), dict(beta=1.0), dict(out=torch.zeros(3, 6)), dict(out=torch.zeros(3, 5).half())):
        with pytest.raises(ValueError):
            ops.adapter_forward(m, **{**good, **bad})
