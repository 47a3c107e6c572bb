"""The paged key/value cache without a GPU: the oracle's closed forms and planted mistakes, the C
entries' refusals (before any launch), the fake kernels' shapes and checks."""
import numpy as np
import pytest
import torch

from cuda_transformer_amd import capi, ops
from oracle import paged
from paged_common import check_attention, f64, make, oracle_attention

OK, INVALID, HEADDIM, LAYOUT = 0, 1, 2, 3


# ----------------------------------------------------------------- the oracle
def dense_attention(q, k, v, scale):
    """Causal attention of the last rows of one sequence by torch, float64: q (n, nh, hs)."""
    n, total = q.shape[0], k.shape[0]
    g = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = torch.einsum("nhd,thd->nht", q, k) * scale
    late = torch.arange(total)[None] > torch.arange(total - n, total)[:, None]
    s = s.masked_fill(late[:, None], -torch.inf)
    return torch.einsum("nht,thd->nhd", s.softmax(-1), v), s.logsumexp(-1)


def sequence(d, b, cache):
    n, ps = int(d["lens"][b]), cache.shape[2]
    rows = [cache[int(d["table"][b, p // ps]), :, p % ps] for p in range(n)]
    return torch.stack(rows).double()


def test_oracle_attention_is_dense_attention():
    d = make(torch.float32, 6, 2, 32, 5, [13, 1, 24], [4, 1, 24])
    O, L, A, dS = oracle_attention(d)
    for b in range(3):
        rows = slice(int(d["cu"][b]), int(d["cu"][b + 1]))
        o, l = dense_attention(d["q"][rows].double(), sequence(d, b, d["k_cache"]),
                               sequence(d, b, d["v_cache"]), 32 ** -0.5)
        np.testing.assert_allclose(O[rows], o, rtol=1e-12, atol=1e-12)
        np.testing.assert_allclose(L[rows], l, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_rotation(interleaved):
    """Norms stay, and scores of rotated rows go by the difference of their positions."""
    rng = np.random.default_rng(0)
    angle = np.arange(40)[:, None] * 0.3 ** np.arange(8)
    q, k = rng.standard_normal((2, 1, 24))
    rot = lambda x, p: paged.rotate(x[None], np.cos(angle[p]), np.sin(angle[p]), interleaved)[0]  # noqa: E731
    np.testing.assert_allclose(np.linalg.norm(rot(q[0], 7)), np.linalg.norm(q[0]))
    np.testing.assert_allclose(rot(q[0], 9) @ rot(k[0], 4), rot(q[0], 35) @ rot(k[0], 30))
    assert (rot(q[0], 9)[16:] == q[0][16:]).all()


def test_planted_mistakes_are_seen():
    """The bounds of the GPU tests are tight enough for the mistakes that such kernels make."""
    d = make(torch.float32, 4, 2, 32, 16, [70, 33], [5, 2], seed=3)
    want = oracle_attention(d)

    def fails(x, scale=None):
        O, L, _, _ = oracle_attention(x, scale)
        with pytest.raises(AssertionError):
            check_attention((torch.from_numpy(O).float(), torch.from_numpy(L).float()), want, torch.float32, 70, 2.0 ** -8)

    O, L, _, _ = want
    check_attention((torch.from_numpy(O).float(), torch.from_numpy(L).float()), want, torch.float32, 70, 0.0)
    filled = {n: torch.nan_to_num(d[n], nan=0.5) for n in ("k_cache", "v_cache")}
    fails(dict(d, **filled, lens=d["lens"] + 1))                   # one key too many
    fails(dict(d, lens=d["lens"] - 1))                             # one too few
    fails(dict(d, **filled, table=d["table"][:, [0, 1, 2, 4, 3]]))  # a last page in front
    fails(dict(d, q=d["q"][:, [1, 0, 2, 3]]))                      # another head
    fails(dict(d, v_cache=d["v_cache"].flip(1)))                   # another kv head
    fails(d, scale=1 / 6.0)


# ----------------------------------------------------------------- refusals at the C boundary
S4, S3 = (2048, 1024, 64, 1), (384, 64, 1)


def c_decode(kc=16, ks=S4, q=16, qs=S3, pages=8, ps=16, P=4, B=2, nh=6, nkv=2, hs=64, scale=0.125, o=16, l=16,
             table=16, lens=16, suffix="", ws=None, ws_bytes=0):
    st = capi.strides
    fn = getattr(capi.lib(), "cta_paged_attention_decode" + suffix)
    return fn(q, st(qs), kc, st(ks), 16, st(S4), pages, ps, table, P, P, lens, B, nh, nkv, hs, scale, o, l, ws, ws_bytes, None)


def c_prefill(N=5, cu=16, B=2, nh=6, q=16, o=16, scale=0.125):
    st = capi.strides
    return capi.lib().cta_paged_attention_prefill(q, st(S3), 16, st(S4), 16, st(S4), 8, 16, 16, 4, 4, 16, cu, B,
                                                  N, nh, 2, 64, scale, o, 16, None, 0, None)


def c_append(N=2, cu=None, rot=0, cos=None, nh=0, q=None, k=16, ks=(128, 64, 1), kcs=S4, hs=64, B=2, q_out=None, nkv=2):
    st = capi.strides
    return capi.lib().cta_paged_kv_append(q, st(S3), k, st(ks), 16, st((128, 64, 1)), N, nh, nkv, hs, cos, cos, rot, 0,
                                          16, st(kcs), 16, st(S4), 8, 16, 16, 4, 4, 16, cu, B, q_out, None)


@pytest.mark.parametrize("kw,code", [
    (dict(hs=48), HEADDIM), (dict(nh=5), INVALID), (dict(nkv=0), INVALID), (dict(ps=0), INVALID),
    (dict(B=-1), INVALID), (dict(P=1 << 28), INVALID), (dict(pages=1 << 31), INVALID),
    (dict(scale=float("nan")), INVALID), (dict(scale=float("inf")), INVALID), (dict(o=None), INVALID),
    (dict(l=None), INVALID), (dict(lens=None), INVALID), (dict(table=None), INVALID),
    (dict(kc=20), LAYOUT), (dict(kc=None), LAYOUT), (dict(q=20), LAYOUT), (dict(o=24), LAYOUT),
    (dict(ks=(2048, 1024, 64, 2)), LAYOUT), (dict(ks=(2048, 1024, 66, 1)), LAYOUT),
    (dict(ks=(2048, 1024, -64, 1)), LAYOUT), (dict(qs=(384, 63, 1)), LAYOUT),
    (dict(ks=(2048, 1024, 68, 1), suffix="_bf16"), LAYOUT), (dict(B=0), OK), (dict(nh=0), OK),
])
def test_decode_refusals(kw, code):
    assert c_decode(**kw) == code
    if code == HEADDIM:
        assert capi.lib().cta_last_error().decode() == (
            "Unsupported head dimension! Only hs=32, hs=64, and hs=128 are supported.")


@pytest.mark.parametrize("kw,code", [
    (dict(cu=None), INVALID), (dict(N=-1), INVALID), (dict(N=(1 << 24) + 1), INVALID), (dict(nh=7), INVALID),
    (dict(q=20), LAYOUT), (dict(o=None), INVALID), (dict(scale=float("nan")), INVALID), (dict(N=0), OK),
])
def test_prefill_refusals(kw, code):
    assert c_prefill(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(N=3), INVALID),                        # no cu_q: one token a sequence
    (dict(rot=8, cos=16, nh=6, q=16, q_out=16), INVALID), (dict(rot=80, cos=16, nh=6, q=16, q_out=16), INVALID),
    (dict(rot=64, nh=6, q=16, q_out=16), LAYOUT), (dict(rot=64, cos=20, nh=6, q=16, q_out=16), LAYOUT),
    (dict(nh=6, q=16), LAYOUT), (dict(nh=6, q=None, q_out=16), LAYOUT), (dict(k=20), LAYOUT),
    (dict(ks=(128, 66, 1)), LAYOUT), (dict(kcs=(2048, 1024, 64, 2)), LAYOUT), (dict(hs=96), HEADDIM),
    (dict(nkv=0), INVALID), (dict(N=1 << 25, B=1 << 25), INVALID), (dict(N=0, B=0), OK), (dict(N=0, cu=16), OK),
])
def test_append_refusals(kw, code):
    assert c_append(**kw) == code


# ----------------------------------------------------------------- the torch layer
def meta(dtype=torch.bfloat16, N=5, B=3, nh=6, nkv=2, hs=64):
    m = dict(device="meta", dtype=dtype)
    i = dict(device="meta", dtype=torch.int32)
    cache = torch.empty(8, nkv, 16, hs, **m)
    return (torch.empty(N, nh, hs, **m), torch.empty(N, nkv, hs, **m), cache,
            torch.empty(B, 4, **i), torch.empty(B, **i), torch.empty(B + 1, **i))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_meta_shapes(dtype):
    q, k, cache, table, lens, cu = meta(dtype)
    O, L = ops.paged_attention_prefill(q, cache, cache, table, lens, cu)
    assert O.shape == q.shape and O.dtype == dtype and L.shape == (5, 6) and L.dtype == torch.float32
    O, L = ops.paged_attention_decode(q[:3], cache, cache, table, lens)
    assert O.shape == (3, 6, 64) and L.shape == (3, 6)
    assert ops.paged_kv_append(k, k, cache, cache, table, lens, cu) is None
    cos = torch.empty(64, 32, device="meta")
    assert ops.paged_kv_append(k, k, cache, cache, table, lens, cu, q, cos, cos).shape == q.shape


def test_fakes_and_wrapper_refuse():
    q, k, cache, table, lens, cu = meta()
    with pytest.raises(Exception):
        ops.paged_attention_decode(q[:3], cache.float(), cache.float(), table, lens)
    with pytest.raises(Exception):
        ops.paged_attention_decode(q[:3], cache, cache, table.long(), lens)
    with pytest.raises(Exception):
        ops.paged_kv_append(k, k, cache, cache, table, lens, cu, q)            # q without cos and sin
    with pytest.raises(Exception):
        ops.paged_kv_append(k, k, cache, cache, table, lens, cu, cos=lens, sin=lens)


def test_no_cpu_fallback():
    d = make(torch.float32, 4, 2, 64, 16, [5], [5])
    with pytest.raises(NotImplementedError):
        ops.paged_attention_prefill(d["q"], d["k_cache"], d["v_cache"], d["table"], d["lens"], d["cu"])
    with pytest.raises(NotImplementedError):
        ops.paged_attention_decode(d["q"][:1], d["k_cache"], d["v_cache"], d["table"], d["lens"])
    with pytest.raises(NotImplementedError):
        ops.paged_kv_append(d["k"], d["v"], d["k_cache"], d["v_cache"], d["table"], d["lens"], d["cu"])


def test_schemas_mark_the_caches_as_written():
    for name in ("paged_kv_append", "paged_kv_append_rotary"):
        schema = str(getattr(torch.ops.cuda_transformer, name).default._schema)
        assert "Tensor(a!) k_cache, Tensor(b!) v_cache" in schema
