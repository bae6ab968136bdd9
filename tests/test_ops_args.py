"""CPU: the 8-bit floating-point Linear operators and the sampler refuse what their kernels do not take (nothing is launched), and
their 64-bit oracle agrees with itself."""
import ctypes

import numpy as np
import pytest
import torch

from cube_amd import hip
from oracle import ops_oracle as oo

P = 0x10000  # a non-null, aligned stand-in pointer: never dereferenced on these paths


def _err(code):
    assert code < 0
    msg = hip.load().cube_last_error().decode()
    assert msg.startswith("cube_"), msg
    return msg


def _fp8(**kw):
    a = hip.Fp8Args(P, 3, 256, P, 8, 8, P, 256, P, 16, 16, 200, P, 0, P, 1, 16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(A=None), dict(W=None), dict(W_scale=None), dict(out=None), dict(A_scale=None), dict(M=-1), dict(N=-1),
                                 dict(K=0), dict(K=(1 << 24) + 1), dict(lda=128), dict(ldw=128), dict(lda=264), dict(ldw=264), dict(lds_a=7),
                                 dict(lds_w=15), dict(ldo=15), dict(out_type=3), dict(out_type=-1), dict(act=3), dict(act=-1), dict(A=P + 8),
                                 dict(W=P + 8), dict(A_scale=P + 2), dict(W_scale=P + 2), dict(bias=P + 2), dict(out=P + 1), dict(a_type=1),
                                 dict(a_type=4)])
def test_gemm_fp8_refuses(bad):
    _err(hip.load().cube_gemm_fp8(ctypes.byref(_fp8(**bad)), None))


@pytest.mark.parametrize("bad", [dict(a_type=3), dict(a_type=-1), dict(lda=199), dict(A=P + 2), dict(A=None), dict(K=0), dict(ldo=3), dict(W=None)])
def test_linear_fp8_refuses(bad):
    lib = hip.load()
    a = _fp8(a_type=0, lda=200, A_scale=None)
    need = lib.cube_linear_fp8_workspace_bytes(a.M, a.N, a.K)
    for k, v in bad.items():
        setattr(a, k, v)
    _err(lib.cube_linear_fp8(ctypes.byref(a), P, max(need, 1 << 20), None))


def test_linear_fp8_refuses_a_workspace_that_is_short():
    lib = hip.load()
    a = _fp8(a_type=0, lda=200, A_scale=None, M=5000, lds_a=5000)
    need = lib.cube_linear_fp8_workspace_bytes(a.M, a.N, a.K)
    assert need > 0
    for ws, n in ((None, need), (P, need - 1), (P + 8, need)):
        _err(lib.cube_linear_fp8(ctypes.byref(a), ws, n, None))


@pytest.mark.parametrize("bad", [dict(x=None), dict(q=None), dict(scale=None), dict(M=-1), dict(K=0), dict(K=(1 << 24) + 1), dict(ld_x=199),
                                 dict(ld_q=255), dict(ld_q=264), dict(ld_s=7), dict(type=3), dict(x=P + 2), dict(q=P + 8), dict(scale=P + 2)])
def test_quant_fp8_refuses(bad):
    a = dict(x=P, type=0, ld_x=200, M=8, K=200, q=P, ld_q=256, scale=P, ld_s=8)
    a.update(bad)
    _err(hip.load().cube_quant_fp8(a["x"], a["type"], a["ld_x"], a["M"], a["K"], a["q"], a["ld_q"], a["scale"], a["ld_s"], None))


@pytest.mark.parametrize("bad", [dict(logits=None), dict(u=None), dict(token=None), dict(M=-1), dict(V=0), dict(V=(1 << 22) + 1), dict(type=3),
                                 dict(ld=99), dict(logits=P + 2), dict(u=P + 4), dict(token=P + 2), dict(prob=P + 2), dict(temperature=P + 1),
                                 dict(top_k=P + 2), dict(top_p=P + 3), dict(min_p=P + 2)])
def test_sample_rows_refuses(bad):
    a = hip.SampleArgs(P, 0, 100, 8, 100, P, None, None, None, None, 1.0, 0, 1.0, 0.0, P, P)
    for k, v in bad.items():
        setattr(a, k, v)
    _err(hip.load().cube_sample_rows(ctypes.byref(a), None, 0, None))


def test_sample_rows_refuses_a_workspace_that_is_short():
    lib = hip.load()
    V = 1 << 20
    a = hip.SampleArgs(P, 0, V, 8, V, P, None, None, None, None, 1.0, 0, 1.0, 0.0, P, P)
    need = lib.cube_sample_workspace_bytes(0, 8, V)
    assert need > 0 and lib.cube_sample_workspace_bytes(0, 8, 200) == 0
    for ws, n in ((None, need), (P, need - 1), (P + 8, need)):
        _err(lib.cube_sample_rows(ctypes.byref(a), ws, n, None))


def test_outputs_over_inputs_and_sizes_past_the_limits_are_refused():
    lib = hip.load()
    far = P + (1 << 32)
    assert "overlaps" in _err(lib.cube_gemm_fp8(ctypes.byref(_fp8()), None))              # out = A
    assert "overlaps" in _err(lib.cube_gemm_fp8(ctypes.byref(_fp8(out=P + 7 * 256 + 254, A=P)), None))   # the last row's last byte
    x = _fp8(a_type=0, lda=200, A_scale=None, out_type=0, ldo=200)
    for out in (P, P + 4 * 199, P + 4 * (200 * 7 + 199), P - 4 * 15):                     # windows of one row distance that meet
        x.out = out
        assert "overlaps" in _err(lib.cube_linear_fp8(ctypes.byref(x), far, 1 << 20, None))
    for kw in (dict(M=(1 << 30) + 1, lds_a=(1 << 30) + 1), dict(N=(1 << 30) + 1, lds_w=(1 << 30) + 1, ldo=1 << 31), dict(ldo=(1 << 40) + 1), dict(ldw=(1 << 24) + 16),
               dict(lda=(1 << 24) + 16)):
        assert "overlaps" not in _err(lib.cube_gemm_fp8(ctypes.byref(_fp8(out=far, **kw)), None))
    assert "lda" in _err(lib.cube_linear_fp8(ctypes.byref(_fp8(a_type=0, lda=(1 << 40) + 1, out=far)), far, 1 << 20, None))
    big = (1 << 30) + 1
    _err(lib.cube_quant_fp8(P, 0, 200, big, 200, far, 256, far, big, None))
    assert lib.cube_linear_fp8_workspace_bytes(big, 16, 200) == 0


def test_null_structures_are_refused():
    lib = hip.load()
    _err(lib.cube_gemm_fp8(None, None))
    _err(lib.cube_linear_fp8(None, None, 0, None))
    _err(lib.cube_sample_rows(None, None, 0, None))


def test_empty_batches_do_nothing():
    lib = hip.load()
    assert lib.cube_gemm_fp8(ctypes.byref(_fp8(M=0, A=None)), None) == 0
    assert lib.cube_gemm_fp8(ctypes.byref(_fp8(N=0, W=None)), None) == 0
    assert lib.cube_linear_fp8(ctypes.byref(_fp8(a_type=0, M=0, A=None)), None, 0, None) == 0
    assert lib.cube_quant_fp8(None, 0, 200, 0, 200, None, 256, None, 0, None) == 0
    a = hip.SampleArgs(None, 0, 100, 0, 100, None, None, None, None, None, 1.0, 0, 1.0, 0.0, None, None)
    assert lib.cube_sample_rows(ctypes.byref(a), None, 0, None) == 0


def test_calls_on_tensors_refuse():
    x = torch.zeros(4, 200)
    with pytest.raises(hip.CubeHipError, match="no CPU fallback"):
        hip.quant_fp8(x)
    with pytest.raises(hip.CubeHipError, match="no CPU fallback"):
        hip.sample_rows(x, torch.zeros(4, dtype=torch.float64))
    for bad in (x.long(), x[0], x.double()):
        with pytest.raises(ValueError):
            hip.quant_fp8(bad)
    rows = hip.Fp8Rows(torch.zeros(4, 256, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.int32), 200)
    with pytest.raises(hip.CubeHipError, match="no CPU fallback"):
        hip.gemm_fp8(rows, rows)
    with pytest.raises(hip.CubeHipError, match="no CPU fallback"):
        hip.linear_fp8(x, rows)
    for q, s, n in ((torch.zeros(4, 200, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.int32), 200),
                    (torch.zeros(4, 256), torch.zeros(1, 4, dtype=torch.int32), 200),
                    (torch.zeros(4, 256, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.int32), 200),
                    (torch.zeros(4, 256, dtype=torch.uint8), torch.zeros(1, 4), 200),
                    (torch.zeros(4, 256, dtype=torch.uint8), torch.zeros(1, 4, dtype=torch.int32), 0),
                    (torch.zeros(4, 512, dtype=torch.uint8)[:, :256], torch.zeros(1, 4, dtype=torch.int32), 200)):
        with pytest.raises(ValueError):
            hip.Fp8Rows(q, s, n)


def test_rows_stand_for_what_the_oracle_says():
    """Fp8Rows.float (torch) against the oracle's decoding of the same bytes, over every code and a range of scales."""
    q = np.arange(256, dtype=np.uint8).reshape(1, 256)
    q = np.concatenate([q, q[:, ::-1], np.zeros_like(q)])
    e = np.array([[127, 130], [100, 140], [0, 254]])
    s = np.zeros((3, 4), dtype=np.uint8)
    s[:, :2] = e
    s = np.ascontiguousarray(s.view(np.int32).T)
    got = hip.Fp8Rows(torch.from_numpy(q.copy()), torch.from_numpy(s), 256).float().numpy()
    v, eb = oo.unpack(q, s, 256)
    np.testing.assert_array_equal(eb, e)
    np.testing.assert_array_equal(got, oo.rows_value(v, eb).astype(np.float32))


@pytest.mark.parametrize("rows,kb", [(3, 1), (1, 1), (1, 5), (5, 4), (5, 6), (0, 2)])
def test_rows_of_any_number_of_scale_words(rows, kb):
    """Fp8Rows.float where the scales are one word a row, one row, or none."""
    rng = np.random.default_rng(rows + kb)
    v = rng.choice(oo.e4m3_values()[:127], (rows, kb * 128))
    e = rng.integers(100, 150, (rows, kb))
    q, s = oo.pack(v, e)
    got = hip.Fp8Rows(torch.from_numpy(q), torch.from_numpy(s), kb * 128).float().numpy()
    np.testing.assert_array_equal(got, oo.rows_value(v, e).astype(np.float32))


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), 1.5, -1])
def test_sampling_refuses_a_limit_that_is_no_count(bad):
    from cube_amd.networks.sampling import Sampling
    with pytest.raises(ValueError):
        Sampling(top_k=bad)


def test_oracle_sampler_against_enumeration():
    """Four candidates by hand: every filter alone, and the empty and greedy rows."""
    z = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    assert [oo.sample_row(z, u)[0] for u in (0.0, 0.39, 0.41, 0.69, 0.71, 0.89, 0.91)] == [1, 1, 3, 3, 2, 2, 0]
    assert [oo.sample_row(z, u, k=2)[0] for u in (0.0, 0.56, 0.58, 0.999)] == [1, 1, 3, 3]
    assert [oo.sample_row(z, u, p=0.6)[0] for u in (0.56, 0.58)] == [1, 3] and oo.sample_row(z, 0.99, p=0.3)[0] == 1
    assert oo.sample_row(z, 0.99, m=0.6)[0] == 3 and oo.sample_row(z, 0.99, m=0.8)[0] == 1
    assert oo.sample_row(z, 0.99, T=0.0)[:2] == (1, 1.0)
    assert oo.sample_row([-np.inf, np.nan], 0.5)[:2] == (-1, 0.0)
    assert oo.sample_row([0.0, -0.0, 0.0], 0.5)[0] == 1
