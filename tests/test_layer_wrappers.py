"""What the tensor wrappers of the layer operators pass on and what they refuse, with a library that only records its calls."""
import pytest
import torch

from hpcdeepneuralnetworks_amd import blas


class OnGpu(torch.Tensor):
    """A host tensor that says it lives on GPU 0; nothing looks at its values."""
    is_cuda = True

    def get_device(self):
        return 0


def gpu(t):
    return t.as_subclass(OnGpu)


def zeros(*shape, dtype=torch.float32):
    return gpu(torch.zeros(*shape, dtype=dtype))


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


@pytest.fixture
def calls(monkeypatch):
    lib = Recorder()
    monkeypatch.setattr(blas._lib, "lib", lambda: lib)
    monkeypatch.setattr(blas, "_device", lambda t, name: 0)
    monkeypatch.setattr(blas, "_stream_of", lambda dev: 0)
    return lib.calls


T, K, C = 6, 2, 8
I32, F32 = torch.int32, torch.float32


def _expert_calls(pos, weights, dweights):
    x, xs = zeros(T, C), zeros(T * K, C)
    yield "pos", lambda: blas.expert_sort(T, K, 4, zeros(T, K, dtype=I32), zeros(5, dtype=I32), pos)
    yield "pos", lambda: blas.expert_gather(T, K, T * K, C, x, pos, xs)
    yield "pos", lambda: blas.expert_combine(T, K, T * K, C, xs, pos, zeros(T, K), x)
    yield "pos", lambda: blas.expert_combine_grad(T, K, T * K, C, x, xs, pos, None, xs, zeros(T, K))
    good = zeros(T, K, dtype=I32)
    yield "weights", lambda: blas.expert_combine(T, K, T * K, C, xs, good, weights, x)
    yield "weights", lambda: blas.expert_combine_grad(T, K, T * K, C, x, xs, good, weights, xs, None)
    yield "dweights", lambda: blas.expert_combine_grad(T, K, T * K, C, x, xs, good, None, xs, dweights)


@pytest.mark.parametrize("shape", [(T, K), (T + 3, K), (T * K,), (T * K + 5,), (1, T, K), (T * K, 1), (1, T * K)])
def test_a_value_per_choice(calls, shape):
    """Rows of topk values without gaps, as the kernels read them, or the same values in one row; more of them may follow."""
    for _, call in _expert_calls(zeros(*shape, dtype=I32), zeros(*shape), zeros(*shape)):
        call()
    assert len(calls) == 7


@pytest.mark.parametrize("shape", [(T, K + 1), (K, T), (T, 2 * K), (T + 1, 1, K + 2), (T - 1, K), (T * K - 1,)])
def test_rows_of_another_length_are_refused(calls, shape):
    for name, call in _expert_calls(zeros(*shape, dtype=I32), zeros(*shape), zeros(*shape)):
        with pytest.raises(blas.HpcdnnError, match=f"^{name} "):
            call()
    assert not calls


def _norm_calls(mean, rstd):
    x, y, good = zeros(T, C), zeros(T, C), zeros(T)
    yield "mean", lambda: blas.layer_norm(T, C, x, None, None, 1e-5, y, mean, good)
    yield "rstd", lambda: blas.layer_norm(T, C, x, None, None, 1e-5, y, good, rstd)
    yield "mean", lambda: blas.layer_norm_grad(T, C, y, x, None, mean, good, zeros(T, C), None, None)
    yield "rstd", lambda: blas.layer_norm_grad(T, C, y, x, None, good, rstd, zeros(T, C), None, None)


@pytest.mark.parametrize("shape", [(T,), (T + 4,), (2, T // 2), (T, 1), (1, T + 1)])
def test_a_value_per_row(calls, shape):
    for _, call in _norm_calls(zeros(*shape), zeros(*shape)):
        call()
    assert len(calls) == 4


@pytest.mark.parametrize("shape", [(T, 2), (2, T), (T + 2, 3), (T - 1,), (2, 2)])
def test_more_than_a_value_per_row_is_refused(calls, shape):
    for name, call in _norm_calls(zeros(*shape), zeros(*shape)):
        with pytest.raises(blas.HpcdnnError, match=f"^{name} "):
            call()
    assert not calls


def _w4(M, N, q, batch=1):
    groups = -(-N // 32)
    return lambda: blas.w4_gemv(batch, M, N, 32, 1.0, q, zeros(M, groups), None, zeros(batch, N), 0.0, zeros(batch, M))


def bytes_(n):
    return torch.zeros(n, dtype=torch.uint8)


@pytest.mark.parametrize("batch", [1, 5])
def test_a_last_row_that_ends_before_its_last_dword_is_refused(calls, batch):
    """Its last dword is read whole: it has to lie in the memory that the tensor stands for."""
    for M, N, q in ((1, 1002, bytes_(501).view(1, 501)), (1, 3, bytes_(2).view(1, 2)), (1, 2, bytes_(1).view(1, 1)),
                    (3, 10, bytes_(2 * 8 + 5).as_strided((3, 5), (8, 1))), (2, 9, bytes_(4 + 8 + 7).as_strided((2, 5), (8, 1), 4)),
                    (1, 9, bytes_(40).view(5, 8)[4:, :5].clone())):
        with pytest.raises(blas.HpcdnnError, match="last row"):
            _w4(M, N, gpu(q), batch)()
    assert not calls


@pytest.mark.parametrize("batch", [1, 5])
def test_a_last_row_inside_its_storage(calls, batch):
    """Narrow views of rows that go on, and rows of whole dwords."""
    cases = ((1, 1002, bytes_(504).view(1, 504)), (1, 1002, bytes_(504).view(1, 504)[:, :501]), (3, 10, bytes_(24).view(3, 8)[:, :5]),
             (1, 9, bytes_(40).view(5, 8)[4:, :5]), (2, 16, bytes_(16).view(2, 8)), (1, 0, bytes_(0).view(1, 0)), (0, 9, bytes_(0).view(0, 5)))
    for M, N, q in cases:
        _w4(M, N, gpu(q), batch)()
    assert len(calls) == len(cases)


@pytest.mark.parametrize("wrong", [1.0, [1.0] * C, "w", object()])
def test_what_is_no_tensor_is_refused_as_everything_else(calls, wrong):
    x, y, v = zeros(T, C), zeros(T, C), zeros(T)
    ids, offsets, pos = zeros(T, K, dtype=I32), zeros(5, dtype=I32), zeros(T, K, dtype=I32)
    q, s = gpu(torch.zeros(4, 4, dtype=torch.uint8)), zeros(4, 1)
    for call in (lambda: blas.layer_norm(T, C, wrong, None, None, 1e-5, y), lambda: blas.layer_norm(T, C, x, None, None, 1e-5, wrong),
                 lambda: blas.layer_norm(T, C, x, wrong, None, 1e-5, y), lambda: blas.layer_norm(T, C, x, None, wrong, 1e-5, y),
                 lambda: blas.layer_norm(T, C, x, None, None, 1e-5, y, wrong, v),
                 lambda: blas.layer_norm_grad(T, C, y, x, None, v, v, None, wrong, None, zeros(99)),
                 lambda: blas.layer_norm_grad(T, C, y, x, None, v, v, None, zeros(C), None, wrong),
                 lambda: blas.w4_gemv(1, 4, 8, 32, 1.0, wrong, s, None, x, 0.0, y), lambda: blas.w4_gemv(1, 4, 8, 32, 1.0, q, wrong, None, x, 0.0, y),
                 lambda: blas.w4_gemv(1, 4, 8, 32, 1.0, q, s, wrong, x, 0.0, y), lambda: blas.w4_gemv(1, 4, 8, 32, 1.0, q, s, None, x, 0.0, wrong),
                 lambda: blas.expert_sort(T, K, 4, wrong, offsets, pos), lambda: blas.expert_sort(T, K, 4, ids, offsets, pos, None, wrong),
                 lambda: blas.expert_sort(T, K, 4, ids, wrong, pos), lambda: blas.expert_gather(T, K, T * K, C, x, wrong, x),
                 lambda: blas.expert_combine(T, K, T, C, x, pos, wrong, y), lambda: blas.expert_combine_grad(T, K, T, C, y, x, pos, None, wrong, None),
                 lambda: blas.w4_quantize(4, 8, 32, wrong, q, s), lambda: blas.w4_quantize(4, 8, 32, x, q, wrong)):
        with pytest.raises(blas.HpcdnnError):
            call()
    assert not calls
