"""Packed attention over the whole range of its types: rows of very different sizes in different tiles and sequences,
values near the ends of the range, gradients of long sequences."""
import math

import pytest
import torch

import attention_plain as plain
from rac_b200 import ext
from test_attention_packed import check, make, run_all

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("r", [1e-3, 1e-4, 1e-5, 1e-6, 1e-8, 1e-30, 0.0])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,small,gain", [([256], slice(128, 256), 1.0), ([256], slice(128, 256), 3.0),
                                             ([256], slice(0, 128), 1.0), ([129], slice(128, 129), 1.0),
                                             ([40, 300, 200], slice(40, 168), 1.0)])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_value_tiles_of_unlike_size(cuda, d, lens, small, gain, causal, r):
    """float32: 128 rows of values, or a last one alone, that are far smaller than the rest of their sequence.  dS of
    their keys holds do . o of the others."""
    q, k, v, go, cu = make(lens, 4, 2, d, F32, cuda, seed=21)
    q = q * gain
    v = v.clone()
    v[small] *= r
    check(run_all(q, k, v, go, cu, causal, d ** -0.5), q, k, v, go, lens, causal, d ** -0.5)


@gpu
@pytest.mark.parametrize("which", ["do", "v", "both"])
def test_tiny_gradients_and_values(cuda, which):
    """float32: do, v or both around 2^-66.  With both, dS lies at the end of the range: 2^-140 is 2^9 of its last
    places, for sums of some 200 terms that are rounded there."""
    lens = [190, 70]
    q, k, v, go, cu = make(lens, 4, 2, 64, F32, cuda, seed=22)
    if which != "v":
        go = go * 2.0 ** -66
    if which != "do":
        v = v * 2.0 ** -66
    got = run_all(q, k, v, go, cu, True, 0.125)
    val, tol = plain.packed(q, k, v, lens, True, 0.125, go)
    for name in ("out", "dq", "dk", "dv"):
        plain.close(got[name], val[name], tol[name] + 2.0 ** -140, name)


@gpu
@pytest.mark.parametrize("d", [64, 128])
def test_gradients_of_long_sequences_keep_their_digits(cuda, d):
    """float32, 32768 rows that all see each other: the weights, and with them dS, are some 2^-15.

    Error of dq and dk, relative to their norm: the tensor core cuts its sums off, at most 2^-23 for each instruction
    of 16 products and in one direction: d / 16 of them for a score, as many for do . v, 8 for a tile of the last
    product; values, weights and dS in 22 bits, 2^-22 each of q, k, v, do, P and dS."""
    n, scale = 32768, d ** -0.5
    q, k, v, go, cu = make([n], 1, 1, d, F32, cuda, seed=23)
    got = run_all(q, k, v, go, cu, False, scale)
    q, k, v, go = (x[:, 0].double() for x in (q, k, v, go))
    dq, dk = torch.zeros_like(q), torch.zeros_like(k)
    for i in range(0, n, 2048):
        sl = slice(i, i + 2048)
        p = torch.softmax(q[sl] @ k.T * scale, 1)
        dp = go[sl] @ v.T
        ds = p * (dp - (p * dp).sum(1, keepdim=True))
        dq[sl] = ds @ k * scale
        dk += ds.T @ q[sl] * scale
    bound = (2 * d / 16 + 8) * 2.0 ** -23 + 6 * 2.0 ** -22
    for name, want in (("dq", dq), ("dk", dk)):
        off = ((got[name][:, 0].double() - want).norm() / want.norm()).item()
        assert off <= bound, (name, off, bound)


@gpu
@pytest.mark.parametrize("size,scale", [(1e-5, 0.0), (1e-20, 0.125), (1e-30, 0.125), (1e-30, -0.125), (1.0, 0.0),
                                        (1e6, 0.0)])
@pytest.mark.parametrize("causal,lens", [(True, [190, 70]), (False, [190, 70])])
def test_scores_of_no_size(cuda, size, scale, causal, lens):
    """float32 queries and keys whose scores vanish: each row is the mean of the values that it sees."""
    q, k, v, go, cu = make(lens, 4, 2, 64, F32, cuda, seed=24)
    q, k = q * size, k * size
    got = run_all(q, k, v, go, cu, causal, scale)
    val, tol = plain.packed(-q if scale < 0 else q, k, v, lens, causal, abs(scale), go)
    if scale < 0:
        val["dq"] = -val["dq"]
    for name in ("out", "dq", "dk", "dv"):
        plain.close(got[name], val[name], tol[name], name)


@gpu
@pytest.mark.parametrize("dt", [F32, F16, BF16])
@pytest.mark.parametrize("other", [2.0 ** 12, math.inf, math.nan])
def test_a_sequence_does_not_feel_the_size_of_another(cuda, dt, other):
    """Gradients of a sequence are the same bits whatever the others hold."""
    lens = [70, 100, 31]
    q, k, v, go, cu = make(lens, 4, 2, 64, dt, cuda, seed=25)
    go = go * 2.0 ** -6
    clean = run_all(q, k, v, go, cu, True, 0.125)
    v, go = v.clone(), go.clone()
    for x in (v, go):
        x[70:170] *= other
    got = run_all(q, k, v, go, cu, True, 0.125)
    for name in ("out", "dq", "dk", "dv"):
        for sl in (slice(0, 70), slice(170, 201)):
            assert torch.equal(got[name][sl], clean[name][sl]), name
    ext.check_device_errors(cuda)
