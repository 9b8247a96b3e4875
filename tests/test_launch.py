"""The short way of a launch with torch tensors (mantle_cuda/_launch): it takes plain calls alone, and
leaves the rest to the long way, which says what is wrong."""
import numpy as np
import pytest
import torch

import mantle_cuda as M
from mantle_cuda import _short

pytest.importorskip("mantle_cuda._launch")  # built with the library where there is torch


def stream():
    return torch.cuda.current_stream().cuda_stream


def short(kernel, args, nd, on=0, scratch=None):
    return M._short_launch(_short(kernel), args, nd, on, scratch)


@pytest.fixture(autouse=True)
def loaded():
    M._with_torch()
    assert M._short_launch is not None


def norm_args(x, y, w, c=64, kind=0, eps=1e-6):
    return (y, None, None, None, x, None, w, c, kind, 0, 0, 0, eps)


def test_what_is_not_plain_is_left_to_the_long_way():
    x, w = torch.zeros(4, 64), torch.zeros(64)
    k = M.kernels.rms_norm
    assert short(k, norm_args(x, x, w), 4) is None                    # on the host
    assert short(k, list(norm_args(x, x, w)), 4) is None              # no tuple
    assert short(k, norm_args(x, x, w)[:-1], 4) is None               # an argument less
    assert short(k, norm_args(M.DevicePtr(256, 1024), x, w), 4) is None
    assert short(k, norm_args(None, None, None), 4) is None           # a buffer the kernel must have
    assert short(k, norm_args(x, x, w), (4,)) is None
    assert short(k, norm_args(x, x, w), 1 << 70) is None
    assert short(k, norm_args(x, x, w), 4, on=-1) is None
    assert short(k, norm_args(x, x, w), 4, on="no") is None
    assert short(k, norm_args(x, x, w, c=1 << 40), 4) is None
    assert short(k, norm_args(x, x, w, kind=0.5), 4) is None
    assert short(k, norm_args(x, x, w, eps=1), 4) is None
    assert short(k, norm_args(x, x, w, eps=1e300), 4) is None
    assert short(k, norm_args(x.to_sparse(), x, w), 4) is None
    assert short(k, norm_args(torch.empty(4, 64, device="meta"), x, w), 4) is None
    with pytest.raises(ValueError):
        M._launch.launch("no plan", (), 1, 0, None)
    with pytest.raises(ValueError, match="fit together"):
        M._launch.plan(0, 0, "BBi", "ff", (1,))
    with pytest.raises(ValueError, match="no such argument"):
        M._launch.plan(0, 0, "BBi", "ff", (-1, 3))


def test_every_kernel_with_operands_has_a_plan():
    for name in M._OPERANDS:
        assert _short(getattr(M.kernels, name)) is not None


@pytest.mark.gpu
def test_plain_calls_take_the_short_way(dev):
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    y, z = torch.empty_like(x), torch.empty_like(x)
    k = M.kernels.rms_norm
    assert short(k, norm_args(x, y, w), 4, stream()) == 0
    k.packed(norm_args(x, z, w), 4, stream())  # the long way
    assert torch.equal(y, z)
    assert short(k, norm_args(torch.nn.Parameter(x), y, w), 4, stream()) == 0
    assert short(k, norm_args(x, y, w), 5, stream()) != 0  # the library's own refusal, as a status
    with pytest.raises(M.ArgumentError, match="the launch touches"):
        M.launch(k, norm_args(x, y, w), 5, stream=stream())
    for bad in (x.half(), x.t().contiguous().t(), x.cpu(), x.to_sparse()):
        assert short(k, norm_args(bad, y, w), 4, stream()) is None
    q, s = torch.empty((4, 64), dtype=torch.uint8, device="cuda"), torch.empty((1, 4), device="cuda")
    for t, fmt, ok in ((torch.uint8, 0, True), (torch.float8_e4m3fn, 0, True), (torch.float8_e5m2, 0, False), (torch.float8_e5m2, 1, True),
                       (torch.float8_e4m3fn, 1, False)):
        got = short(k, (y, q.view(t), s, None, x, None, w, 64, 0, 0, fmt, 0, 1e-6), 4, stream())
        assert got == (0 if ok else None)
    args = (y, w, x, x, w, None, 64, 0, 0, 1e-6)
    need = M.workspace_bytes(M.kernels.rms_norm_grad, args, 4)
    assert short(M.kernels.rms_norm_grad, args, 4, stream(), torch.empty(need, dtype=torch.uint8, device="cuda")) == 0
    assert short(M.kernels.rms_norm_grad, args, 4, stream(), torch.empty(need, dtype=torch.uint8)) is None
    assert short(M.kernels.rms_norm_grad, args, 4, stream()) not in (0, None)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_a_tensor_without_storage_is_refused(dev):
    from torch._subclasses.fake_tensor import FakeTensorMode
    x, w = torch.randn(4, 64, device="cuda"), torch.ones(64, device="cuda")
    with FakeTensorMode():
        fake = torch.empty(4, 64, device="cuda")
    assert short(M.kernels.rms_norm, norm_args(fake, x, w), 4, stream()) is None


@pytest.mark.gpu
def test_buffers_take_the_long_way_to_the_same_results(dev):
    r, c = 70, 333
    h, dy, w = torch.randn(r, c, device="cuda"), torch.randn(r, c, device="cuda"), torch.randn(c, device="cuda")
    dx, dw = torch.empty_like(h), torch.empty_like(w)
    k = M.kernels.rms_norm_grad
    args = (dx, dw, dy, h, w, None, c, 0, 0, 1e-6)
    need = M.workspace_bytes(k, args, r)
    M.launch(k, args, r, stream=stream(), workspace=torch.empty(need, dtype=torch.uint8, device="cuda"))
    torch.cuda.synchronize()
    B = lambda t: M.Buffer(dev, t.cpu().numpy().reshape(-1))  # noqa: E731
    DX, DW, ws = M.Buffer(dev, np.float32, r * c), M.Buffer(dev, np.float32, c), M.Buffer(dev, np.uint8, need)
    bufs = (DX, DW, B(dy), B(h), B(w), None, c, 0, 0, 1e-6)
    assert M.workspace_bytes(k, bufs, r) == need
    M.launch(k, bufs, r, stream=dev.stream, workspace=ws)
    dev.synchronize()
    assert np.array_equal(DX.array(), dx.cpu().numpy().reshape(-1)) and np.array_equal(DW.array(), dw.cpu().numpy())
    with pytest.raises(M.ArgumentError, match="of scratch"):
        M.launch(k, bufs, r, stream=dev.stream)
    with pytest.raises(M.ArgumentError, match="of scratch"):
        M.launch(k, bufs, r, stream=dev.stream, workspace=M.Buffer(dev, np.uint8, need - 4))
    with pytest.raises(M.ArgumentError, match="h: "):
        M.launch(k, (DX, DW, B(dy), DW, B(w), None, c, 0, 0, 1e-6), r, stream=dev.stream, workspace=ws)
    with pytest.raises(M.ArgumentError, match="expected Float32"):
        M.launch(k, (DX, ws, B(dy), B(h), B(w), None, c, 0, 0, 1e-6), r, stream=dev.stream, workspace=ws)


@pytest.mark.gpu
def test_launches_from_threads_at_once(dev):
    # the launch runs without the interpreter's lock: each thread its own results, refusals and streams
    import threading
    k, errors = M.kernels, []
    cases = [(5 + i, 64 * (i + 1)) for i in range(6)]
    data = [(torch.randn(r, c, device="cuda"), torch.ones(c, device="cuda")) for r, c in cases]
    want = [torch.empty_like(x) for x, _ in data]
    for (x, w), y, (r, c) in zip(data, want, cases):
        M.launch(k.rms_norm, norm_args(x, y, w, c=c), r, stream=stream())
    torch.cuda.synchronize()

    def work(i):
        try:
            (x, w), (r, c) = data[i], cases[i]
            side, y = torch.cuda.Stream(), torch.empty_like(x)
            dx, dw = torch.empty_like(x), torch.empty_like(w)
            grad = (dx, dw, x, x, w, None, c, 0, 0, 1e-6)
            ws = torch.empty(M.workspace_bytes(k.rms_norm_grad, grad, r), dtype=torch.uint8, device="cuda")
            side.wait_stream(torch.cuda.current_stream())
            for _ in range(100):
                M.launch(k.rms_norm, norm_args(x, y, w, c=c), r, stream=side.cuda_stream)
                M.launch(k.rms_norm_grad, grad, r, stream=side.cuda_stream, workspace=ws)
                with pytest.raises(M.ArgumentError, match=f"y: {4 * r * c} bytes, the launch touches {4 * (r + 1) * c}"):
                    M.launch(k.rms_norm, norm_args(x, y, w, c=c), r + 1, stream=side.cuda_stream)
            side.synchronize()
            assert torch.equal(y, want[i])
        except BaseException as e:
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
