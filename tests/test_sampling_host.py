"""Refusals of sampling that need no GPU, and the C ABI's own checks (no kernel is launched)."""

import pytest

from kernel_optim_amd import _lib
from kernel_optim_amd.kernels import sampling as S


@pytest.mark.parametrize("B,V,device", [(0, 8, "cuda:0"), (65536, 8, "cuda:0"), (1, 0, "cuda:0"),
                                        (1, (1 << 20) + 1, "cuda:0"), (1, 8, "cpu")])
def test_sampler_refuses(B, V, device):
    with pytest.raises(ValueError):
        S.Sampler(B, V, device)


def test_chunks():
    for B in (1, 2, 64, 300, 65535):
        for V in (1, 4096, 4097, 151936, 1 << 20):
            c = S._chunks(B, V)
            assert 1 <= c <= 1024 and (c == 1 or B * c <= 512)


def test_c_abi_refuses():
    h, p = _lib.lib(), 1 << 20   # p is never read: the checks come first
    EINVAL, ERANGE = -22, -34

    def call(x=p, f32=0, stride=8, B=1, V=8, u=p, ids=p, scratch=p, n=1 << 20, chunks=2):
        return h.ko_sample(x, f32, stride, B, V, u, None, 1.0, None, 0, None, 1.0, None, 0.0, ids,
                           None, scratch, n, chunks, None)

    assert call(x=None) == call(u=None) == call(ids=None) == call(scratch=None) == EINVAL
    assert call(x=p + 1) == call(x=p + 2, f32=1) == call(scratch=p + 8) == EINVAL
    assert call(B=0) == call(V=0) == call(stride=-1) == call(chunks=0) == EINVAL
    assert call(n=h.ko_sample_scratch(1, 2) - 1) == EINVAL
    assert call(V=(1 << 20) + 1) == call(B=65536) == call(chunks=1025) == ERANGE
    assert h.ko_sample_scratch(0, 1) == h.ko_sample_scratch(1, 0) == h.ko_sample_scratch(1, 1025) == -1
    assert h.ko_sample_scratch(7, 1) == 0


def test_engine_settings():
    from kernel_optim_amd.engine import Sampling
    t, k, p, m = Sampling(temperature=[0.5, 1], top_k=2 ** 40, top_p=0.25).columns(2)
    assert t.tolist() == [0.5, 1.0] and k.tolist() == [2 ** 31 - 1] * 2
    assert p.tolist() == [0.25, 0.25] and m.tolist() == [0.0, 0.0]
    for bad in (Sampling(temperature=-1), Sampling(top_k=1.5), Sampling(top_p=2), Sampling(min_p="0"),
                Sampling(temperature=[1.0]), Sampling(min_p=float("nan"))):
        with pytest.raises(ValueError):
            bad.columns(2)


@pytest.mark.parametrize("k", [float("inf"), float("nan"), 2.5, -1])
def test_top_k_is_a_whole_number(k):
    from kernel_optim_amd.engine import Sampling
    with pytest.raises(ValueError):
        Sampling(top_k=k).columns(1)
    with pytest.raises(ValueError):
        S._setting(k, "top_k", None, 1, 0, S._whole)
