"""Inputs and error bounds shared by the tests of the paged key/value cache."""
import numpy as np
import torch

from oracle import paged

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def make(dtype, nh, nkv, hs, ps, lens, news=None, seed=0, spare=2, width=None, holes=(), scale=1.0,
         garbage=float("nan"), device="cpu"):
    """A cache of sequences of `lens` tokens, the last `news` of them new (default: one each, none
    for an empty one).  Pages are shuffled; every row that holds no token is `garbage`, and so are
    `spare` unmapped pages.  holes: (sequence, page index) entries of the table set to -1."""
    g = torch.Generator().manual_seed(seed)
    news = [min(n, 1) for n in lens] if news is None else list(news)
    used = [-(-n // ps) for n in lens]
    width = max(used + [1]) if width is None else width
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for b, u in enumerate(used):
        table[b, :u] = torch.tensor(order[at:at + u], dtype=torch.int32)
        at += u
    caches = []
    for _ in range(2):
        c = torch.randn(pages, nkv, ps, hs, generator=g) * scale
        live = torch.zeros(pages, ps, dtype=torch.bool)
        for b, n in enumerate(lens):
            for i in range(used[b]):
                live[table[b, i], :max(0, min(ps, n - i * ps))] = True
        c = torch.where(live[:, None, :, None], c, garbage)
        caches.append(c.to(dtype))
    for b, i in holes:
        table[b, i] = -1
    cu = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    n = int(cu[-1])
    q, k, v = ((torch.randn(n, h, hs, generator=g) * scale).to(dtype) for h in (nh, nkv, nkv))
    d = dict(q=q, k=k, v=v, k_cache=caches[0], v_cache=caches[1], table=table,
             lens=torch.tensor(lens, dtype=torch.int32), cu=torch.from_numpy(cu))
    return {name: t.to(device) for name, t in d.items()}


def f64(t):
    return t.detach().cpu().double().numpy()


def oracle_attention(d, scale=None, cu=None):
    """The oracle on make()'s tensors; rows that hold no token may be garbage."""
    hs = d["q"].shape[-1]
    return paged.attention(f64(d["q"]), f64(d["k_cache"]), f64(d["v_cache"]), d["table"].cpu().tolist(),
                           d["lens"].cpu().tolist(), (d["cu"] if cu is None else cu).cpu().tolist(),
                           hs ** -0.5 if scale is None else scale)


U = 2.0 ** -24  # half a step of FP32, relative


def check_attention(got, want, dtype, n_keys, p_round):
    """(O, L) against the oracle's (O, L, A, dS), with what FP32 arithmetic allows.

    A score is a sum of hs products in any order and two roundings (the scale, the exponent's
    difference): off by at most (hs + 2) u dS, and 2 u max|s| <= 2 u dS: ds in all.  exp2 is good
    to 2^-22, so a probability is off by ds + 2^-22, relative.  O = (sum p v) / (sum p), n terms
    each in any order, a quotient and at most 4 rescalings of partial sums: relative to
    A = sum p |v| / l twice (ds + 2^-22 + n u) + 8 u, and p_round where P is rounded as a matrix
    operand; then O's own rounding, eps/2 of its type, and half of its smallest number.
    ln(sum p): ds + 2^-22 + n u, the logarithm and the sum 4 u of their values."""
    O, L = got
    O_ref, L_ref, A, dS = want
    hs = O.shape[-1]
    assert O.dtype == dtype and L.dtype == torch.float32
    assert O.shape == O_ref.shape and L.shape == L_ref.shape
    O, L = f64(O), f64(L)
    rel = (hs + 4) * U * dS + 2.0 ** -22 + n_keys * U
    tol = A * (2 * rel + 8 * U + p_round)[..., None] + np.abs(O_ref) * torch.finfo(dtype).eps / 2
    tol += torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = np.abs(O - O_ref)
    assert not np.isnan(O).any(), "NaN in O"
    assert (off <= tol).all(), f"O: {(off / tol).max():.3g} of the bound, {off.max():.3g} off"
    empty = np.isinf(L_ref)
    assert (np.isneginf(L) == empty).all()
    assert (O[empty] == 0).all()
    off = np.abs(L[~empty] - L_ref[~empty])
    tol = (rel + 4 * U * (np.abs(np.where(empty, 0, L_ref)) + np.log(n_keys + 1)))[~empty]
    assert (off <= tol).all(), f"L: {(off / tol).max():.3g} of the bound"
