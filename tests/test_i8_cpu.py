"""What the 8-bit rows, their projections and the scores of tokens refuse, as far as it is decided before a GPU is asked."""
import ctypes as C

import pytest
import torch

from ferrum_b200 import _lib, surface as s

F32 = torch.float32


class Library:
    def __getattr__(self, name):
        def call(*args):
            raise AssertionError(name + " was called")
        return call


class Handle:
    """A device handle whose library must not be called; its tensors lie on the CPU (ordinal -1) or on the GPU that is not there."""
    handle, _L = None, Library()

    def __init__(self, ordinal):
        self.ordinal, self.torch_device = ordinal, torch.device("cuda", max(ordinal, 0))

    def check(self, rc):
        raise AssertionError("the library was called")


class Weights:
    rows, cols, handle = 8, 32, C.c_void_p(1)


def rows(n=32, count=4):
    return torch.zeros(count, n), torch.zeros(count, n, dtype=torch.int8), torch.zeros(count)


def calls(d):
    x, q, sc = rows()
    w, y, ids = torch.ones(32), torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32)
    return {"quantize": lambda: s.quantize_i8(d, x, 4, q, sc), "rmsnorm": lambda: s.rmsnorm_i8(d, x, w, 1e-6, 4, q, sc),
            "add": lambda: s.add_rmsnorm_i8(d, x, x, w, 1e-6, 4, x, q, sc), "glu": lambda: s.glu_i8(d, x, x, 4, q, sc),
            "project": lambda: s.project_i8(d, Weights, q, sc, 4, y), "many": lambda: s.project_many_i8(d, [Weights], q, sc, 4, [y]),
            "scores": lambda: s.token_logprobs(d, x, 32, 4, ids, sc, None, None)}


@pytest.mark.parametrize("name", calls(None))
def test_tensors_that_are_not_on_the_handles_device(name):
    with pytest.raises(s.DeviceMismatch):
        calls(Handle(0))[name]()


def test_rows_refused():
    d = Handle(-1)
    x, q, sc = rows()
    w = torch.ones(32)
    for call, error in ((lambda: s.quantize_i8(d, x, 0, q, sc), s.ShapeError), (lambda: s.quantize_i8(d, x, 3, q, sc), s.ShapeError),
                        (lambda: s.quantize_i8(d, x, -4, q, sc), s.ShapeError), (lambda: s.quantize_i8(d, x, 4, q[:3], sc), s.ShapeError),
                        (lambda: s.quantize_i8(d, x, 4, q, sc[:3]), s.ShapeError), (lambda: s.quantize_i8(d, x, 4, q.int(), sc), s.Unsupported),
                        (lambda: s.quantize_i8(d, x, 4, q, sc.double()), s.Unsupported), (lambda: s.quantize_i8(d, x.t(), 4, q, sc), s.ShapeError),
                        (lambda: s.rmsnorm_i8(d, x, w[:31], 1e-6, 4, q, sc), s.ShapeError), (lambda: s.rmsnorm_i8(d, x, w.bfloat16(), 1e-6, 4, q, sc), s.Unsupported),
                        (lambda: s.add_rmsnorm_i8(d, x, x[:3], w, 1e-6, 4, x, q, sc), s.ShapeError),
                        (lambda: s.add_rmsnorm_i8(d, x, x.bfloat16(), w, 1e-6, 4, x, q, sc), s.Unsupported),
                        (lambda: s.add_rmsnorm_i8(d, x, x, w, 1e-6, 4, x.bfloat16(), q, sc), s.Unsupported),
                        (lambda: s.glu_i8(d, x, x.bfloat16(), 4, q, sc), s.Unsupported), (lambda: s.glu_i8(d, x, x[:3], 4, q, sc), s.ShapeError)):
        with pytest.raises(error):
            call()


def test_more_rows_than_the_interface_counts():
    """Sizes that 32 bits would cut to others are refused, not cut."""
    d = Handle(-1)

    class Flat:  # a contiguous tensor of that many values, without their memory
        def __init__(self, dtype, count):
            self.dtype, self.count = dtype, count

        def numel(self):
            return self.count

        def get_device(self):
            return -1

        def is_contiguous(self):
            return True
    with pytest.raises(s.ShapeError):
        s.quantize_i8(d, Flat(F32, 2 ** 32 + 4), 1, Flat(torch.int8, 2 ** 32 + 4), torch.zeros(1))
    with pytest.raises(s.ShapeError):
        s.quantize_i8(d, Flat(F32, 4 * (2 ** 32 + 1)), 2 ** 32 + 1, Flat(torch.int8, 4 * (2 ** 32 + 1)), Flat(F32, 2 ** 32 + 1))
    with pytest.raises(s.ShapeError):
        s.token_logprobs(d, Flat(F32, 2 ** 32 + 4), 2 ** 32 + 4, 1, None, None, None, torch.zeros(1))


def test_projections_refused():
    d = Handle(-1)
    _, q, sc = rows()
    y = torch.zeros(4, 8)
    for call, error in ((lambda: s.project_i8(d, Weights, q.int(), sc, 4, y), s.Unsupported), (lambda: s.project_i8(d, Weights, q, sc[:3], 4, y), s.ShapeError),
                        (lambda: s.project_many_i8(d, [], q, sc, 4, []), s.ParameterError), (lambda: s.project_many_i8(d, [Weights], q, sc, 4, [y, y]), s.ParameterError),
                        (lambda: s.project_many_i8(d, [Weights], q, sc, 4, [y[:3]]), s.ShapeError),
                        (lambda: s.project_many_i8(d, [Weights, Weights], q, sc, 4, [y, y.bfloat16()]), s.Unsupported)):
        with pytest.raises(error):
            call()
    for values, scales, error in ((torch.zeros(8, 32), torch.zeros(8), s.Unsupported), (torch.zeros(8, 32, dtype=torch.int8), torch.zeros(7), s.ShapeError),
                                  (torch.zeros(8, dtype=torch.int8), torch.zeros(8), s.ShapeError), (torch.zeros(32, 8, dtype=torch.int8).t(), torch.zeros(8), s.ShapeError),
                                  (torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8, dtype=torch.float64), s.Unsupported)):
        with pytest.raises(error):
            s.Matrix.from_i8(d, values, scales)


def test_scores_refused():
    d = Handle(-1)
    l, ids, lp = torch.zeros(4, 100), torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    for call, error in ((lambda: s.token_logprobs(d, l, 0, 4, ids, lp, None, None), s.ShapeError), (lambda: s.token_logprobs(d, l, 100, 0, ids, lp, None, None), s.ShapeError),
                        (lambda: s.token_logprobs(d, l, 101, 4, ids, lp, None, None), s.ShapeError), (lambda: s.token_logprobs(d, l, 100, 4, ids, lp, None, None, stride=99), s.ShapeError),
                        (lambda: s.token_logprobs(d, l, 100, 4, ids, lp, None, None, stride=101), s.ShapeError), (lambda: s.token_logprobs(d, l, 100, 4, ids.long(), lp, None, None), s.Unsupported),
                        (lambda: s.token_logprobs(d, l, 100, 4, ids, lp, None, None, -1), s.ParameterError), (lambda: s.token_logprobs(d, l, 100, 4, ids, lp, None, None, 2 ** 32), s.ParameterError),
                        (lambda: s.token_logprobs(d, l, 100, 4, ids, lp, None, None, 2, torch.zeros(4, 3), torch.zeros(4, 2, dtype=torch.int32)), s.ShapeError)):
        with pytest.raises(error):
            call()


def test_null_handles_are_errors():
    lib = _lib.load()
    out = C.c_void_p()
    assert lib.fq_quantize_i8(None, None, _lib.F32, 4, 1, None, None) == _lib.ERR_PARAM
    assert lib.fq_rmsnorm_i8(None, None, _lib.F32, None, 4, 1e-6, 1, None, None) == _lib.ERR_PARAM
    assert lib.fq_add_rmsnorm_i8(None, None, None, _lib.F32, None, 4, 1e-6, 1, None, None, None) == _lib.ERR_PARAM
    assert lib.fq_glu_i8(None, None, None, _lib.F32, 4, 1, None, None) == _lib.ERR_PARAM
    assert lib.fq_matrix_create_i8(None, 1, 16, None, None, C.byref(out)) == _lib.ERR_PARAM and not out.value
    assert lib.fq_project_i8(None, None, None, 16, None, 1, None, _lib.F32, 1) == _lib.ERR_PARAM
    assert lib.fq_project_many_i8(None, None, 1, None, 16, None, 1, None, _lib.F32) == _lib.ERR_PARAM
    assert lib.fq_token_logprobs(None, None, _lib.F32, 4, 4, 1, None, 0, None, None, None, None, None) == _lib.ERR_PARAM
