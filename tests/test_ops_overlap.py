"""CPU: the 8-bit Linear operators and the sampler refuse an output or a workspace over anything that the call reads (nothing is launched
on these paths), and take memory that only lies beside it -- up to the refusal that follows."""
import ctypes
import random

import pytest

from cube_amd import hip

MB = 1 << 20


def refused(code):
    assert code < 0
    return hip.load().cube_last_error().decode()


def fp8(**kw):
    """8 x 16 outputs of K = 200, every array in a megabyte of its own."""
    a = hip.Fp8Args(1 * MB, 3, 256, 2 * MB, 8, 8, 3 * MB, 256, 4 * MB, 16, 16, 200, 5 * MB, 0, 6 * MB, 1, 16)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


SIZES = {"A": (1 * MB, 8 * 256), "A_scale": (2 * MB, 8 * 4), "W": (3 * MB, 16 * 256), "W_scale": (4 * MB, 16 * 4), "bias": (5 * MB, 16 * 4)}


@pytest.mark.parametrize("name", list(SIZES))
def test_gemm_fp8_refuses_out_over(name):
    at, size = SIZES[name]
    for out in (at, at + size - 2, at - 8 * 16 * 2 + 2):       # on its first byte, its last two, ending two bytes into it
        assert refused(hip.load().cube_gemm_fp8(ctypes.byref(fp8(out=out)), None)).endswith("out overlaps " + name)


@pytest.mark.parametrize("name", ["A", "W", "W_scale", "bias"])
def test_linear_fp8_refuses_out_and_workspace_over(name):
    lib = hip.load()
    M = 100
    a = fp8(a_type=0, lda=200, A_scale=None, M=M)
    need = lib.cube_linear_fp8_workspace_bytes(M, 16, 200)
    assert need > 0
    at, size = SIZES[name][0], {"A": M * 800}.get(name, SIZES[name][1])
    for out in (at, at + size - 2):
        a.out = out
        assert refused(lib.cube_linear_fp8(ctypes.byref(a), 8 * MB, need, None)).endswith("out overlaps " + name)
    a.out = 6 * MB
    for ws in (at, (at + size - 1) // 16 * 16, at - need // 16 * 16 + 16):
        assert refused(lib.cube_linear_fp8(ctypes.byref(a), ws, need, None)).endswith("the workspace overlaps " + name)
    assert refused(lib.cube_linear_fp8(ctypes.byref(a), 6 * MB + 16, need, None)).endswith("the workspace overlaps out")


def test_quant_fp8_refuses_its_arrays_over_one_another():
    f = hip.load().cube_quant_fp8
    x, q, s = 1 * MB, 2 * MB, 3 * MB
    for kw in (dict(q=x), dict(q=x + 8 * 800 - 16), dict(s=x), dict(s=x + 8 * 800 - 4), dict(s=q), dict(s=q + 8 * 256 - 4), dict(q=s)):
        p = dict(x=x, q=q, s=s)
        p.update(kw)
        assert "overlap" in refused(f(p["x"], 0, 200, 8, 200, p["q"], 256, p["s"], 8, None))


@pytest.mark.parametrize("V,ws", [(100, False), (1 << 20, True)])
def test_sample_rows_refuses_outputs_over(V, ws):
    lib = hip.load()
    M = 8
    need = lib.cube_sample_workspace_bytes(0, M, V)
    assert (need > 0) == ws
    big = 1 << 30
    at = dict(logits=1 * big, u=2 * big, temperature=3 * big, top_k=4 * big, top_p=5 * big, min_p=6 * big, token=7 * big, prob=8 * big)
    size = dict(logits=M * V * 4, u=M * 8)

    def call(w=9 * big, **kw):
        p = dict(at)
        p.update(kw)
        a = hip.SampleArgs(p["logits"], 0, V, M, V, p["u"], p["temperature"], p["top_k"], p["top_p"], p["min_p"], 0, 0, 0, 0, p["token"], p["prob"])
        return refused(lib.cube_sample_rows(ctypes.byref(a), w if ws else None, need, None))

    for name in ("logits", "u", "temperature", "top_k", "top_p", "min_p"):
        for out in ("token", "prob"):
            assert "overlap" in call(**{out: at[name]}) and "overlap" in call(**{out: at[name] + size.get(name, 4 * M) - 4})
        if ws:
            assert "overlap" in call(w=at[name])
    assert "overlap" in call(token=at["prob"] + 4 * M - 4)
    if ws:
        assert "overlap" in call(w=at["prob"]) and "overlap" in call(w=at["token"])


def test_areas_against_their_bytes():
    """Random small layouts of cube_quant_fp8 (f32 rows, codes, scales) that share a byte by the sets of their bytes are all refused.  (That
    the others are taken is for the GPU: tests/test_gpu_fp8_more.py.)"""
    rng = random.Random(1)
    f = hip.load().cube_quant_fp8
    hits = 0
    for _ in range(3000):
        M, K = rng.randint(1, 6), rng.randint(1, 140)
        kb = -(-K // 128)
        ld_x, ld_q, ld_s = K + rng.choice([0, 0, 5, 300]), kb * 128 + 16 * rng.choice([0, 0, 1, 9]), M + rng.choice([0, 3])
        x = MB + 4 * rng.randint(0, 400)
        q = MB + 16 * rng.randint(0, 300)
        s = 8 * MB if rng.random() < 0.5 else MB + 4 * rng.randint(0, 1200)
        bx = {x + 4 * ld_x * r + i for r in range(M) for i in range(4 * K)}
        bq = {q + ld_q * r + i for r in range(M) for i in range(kb * 128)}
        bs = {s + i for i in range(4 * M)}
        if bx & bq or bx & bs or bq & bs:
            hits += 1
            assert "overlap" in refused(f(x, 0, ld_x, M, K, q, ld_q, s, ld_s, None)), (x, ld_x, M, K, q, ld_q, s, ld_s)
    assert hits > 500


def test_sample_rows_refuses_a_row_distance_whose_bytes_overflow():
    a = hip.SampleArgs(1 * MB, 0, 1 << 62, 8, 100, 2 * MB, None, None, None, None, 1.0, 0, 1.0, 0.0, 3 * MB, 4 * MB)
    assert "ld=" in refused(hip.load().cube_sample_rows(ctypes.byref(a), None, 0, None))
