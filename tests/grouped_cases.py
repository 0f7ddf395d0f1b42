"""Shared by the tests of the grouped and the 4-bit products: storage of the element types, a 64-bit
statement of the grouped products, and tolerances.

Tolerance of an accumulated element, term by term: the products of two 16-bit (or 4-bit) values are exact
in binary32; each of the at most K + 2 additions that follow (the accumulation and beta * C) is off by at
most one unit in the last place, 2^-23, of a partial sum that is no larger than S = |alpha| sum|a||b| +
|beta c|; the scaling by alpha and beta adds 2 * 2^-24 of the same S.  So |d - exact| <= (K + 3) 2^-23 S,
and a 16-bit result adds half a step of its own: eps/2 |d| or half the smallest subnormal."""
import numpy as np

from cudanative_jl_b200.bfloat16 import BFloat16, round_to_bf16, widen_bf16

HALF_STEP = {np.float32: (2.0 ** -24, 2.0 ** -150), np.float16: (2.0 ** -11, 2.0 ** -25), BFloat16: (2.0 ** -8, 2.0 ** -134)}


def store(x, elem):
    """Values -> the array as it lies in memory."""
    x = np.asarray(x, dtype=np.float32)
    return np.asfortranarray(round_to_bf16(x) if elem is BFloat16 else x.astype(elem))


def value(x, elem):
    return (widen_bf16(x) if elem is BFloat16 else x).astype(np.float64)


def memory_type(elem):
    return np.uint16 if elem is BFloat16 else np.dtype(elem)


def offsets_of(sizes, start=0):
    return (start + np.concatenate([[0], np.cumsum(sizes)])).astype(np.int32)


def close(got, exact, S, K, elem, what=""):
    """got: values read back (float64); exact and S as above; NaN and infinities must be where exact has them."""
    rel, tiny = HALF_STEP[elem]
    with np.errstate(invalid="ignore", over="ignore"):
        tol = (K + 3) * 2.0 ** -23 * S
        tol = tol + rel * (np.abs(exact) + tol) + tiny
        finite = np.isfinite(exact)
        assert np.array_equal(np.isfinite(got), finite), f"{what}: non-finite values differ"
        off = np.where(finite, np.abs(got - exact) - tol, 0.0)
    at = np.unravel_index(int(np.argmax(off)), off.shape) if off.size else None
    assert off.size == 0 or off[at] <= 0, f"{what}: at {at} {got[at]} instead of {exact[at]}, tolerance {tol[at]}"


def grouped_ref(A, B, C, offsets, alpha, beta, transA, D):
    """A: list of stored matrices per group, in float64.  Returns exact D, S; columns of no group are D's."""
    exact, S = D.copy(), np.zeros(D.shape)
    for e, a in enumerate(A):
        s = slice(int(offsets[e]), int(offsets[e + 1]))
        op = a.T if transA else a
        exact[:, s] = alpha * (op @ B[:, s])
        S[:, s] = abs(alpha) * (np.abs(op) @ np.abs(B[:, s]))
        if beta:
            exact[:, s] += beta * C[:, s]
            S[:, s] += np.abs(beta * C[:, s])
    return exact, S


def grouped_k_ref(A, B, C, offsets, alpha, beta):
    """A (M x K), B (N x K), C list of M x N or None, in float64: lists of exact D_e and S_e."""
    exact, S = [], []
    for e in range(len(offsets) - 1):
        s = slice(int(offsets[e]), int(offsets[e + 1]))
        d, t = alpha * (A[:, s] @ B[:, s].T), abs(alpha) * (np.abs(A[:, s]) @ np.abs(B[:, s].T))
        if beta:
            d, t = d + beta * C[e], t + np.abs(beta * C[e])
        exact.append(d)
        S.append(t)
    return exact, S
