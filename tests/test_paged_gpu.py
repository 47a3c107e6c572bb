"""The paged key/value cache on the GPU against the float64 oracle: appending (with and without the
rotation), attention of one new token a sequence, attention of packed new tokens."""
import numpy as np
import pytest
import torch

from cuda_transformer_amd import ops
from oracle import paged
from paged_common import DTYPES, check_attention, f64, make, oracle_attention

pytestmark = pytest.mark.gpu

ALL = list(DTYPES)


def to(d, device):
    return {k: t.to(device) for k, t in d.items()}


def p_round_decode(dtype):
    """One-token attention keeps a probability's two leading parts (16 bits and more)."""
    return 0.0 if dtype == torch.float32 else 2.0 ** -16


def p_round_prefill(dtype):
    """Probabilities are rounded once to the type of V as a matrix operand."""
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def run_decode(d, cuda, scale=None):
    g = to(d, cuda)
    return ops.paged_attention_decode(g["q"], g["k_cache"], g["v_cache"], g["table"], g["lens"], scale)


def check_decode(d, cuda, scale=None):
    B = d["lens"].numel()
    cu = torch.arange(B + 1, dtype=torch.int32)
    got = run_decode(d, cuda, scale)
    n = max(1, int(d["lens"].clamp(0, d["table"].shape[1] * d["k_cache"].shape[2]).max()))
    check_attention(got, oracle_attention(d, scale, cu), d["q"].dtype, n, p_round_decode(d["q"].dtype))
    return got


def decode_inputs(dtype, nh, nkv, hs, ps, lens, **kw):
    """One query a sequence, empty ones included."""
    return make(DTYPES[dtype], nh, nkv, hs, ps, lens, news=[1] * len(lens), **kw)


# ----------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("hs,nh,nkv,ps,rot,interleaved,lens,news", [
    (64, 6, 6, 16, 0, False, [1, 17, 200], [1, 1, 1]),
    (64, 6, 6, 16, 64, False, [1, 17, 200], [1, 1, 1]),
    (128, 8, 2, 7, 128, True, [5, 40, 33], [5, 3, 0]),
    (128, 12, 4, 32, 64, False, [33, 0, 64, 1], [33, 0, 31, 1]),
    (32, 3, 1, 1, 16, True, [9, 2], [4, 2]),
    (32, 4, 2, 100, 32, False, [130] * 70, [2] * 70),   # more sequences than a wave's lanes
    (64, 1, 1, 24, 32, False, [300, 257], [300, 1]),
])
def test_append(cuda, dtype, hs, nh, nkv, ps, rot, interleaved, lens, news):
    dt = DTYPES[dtype]
    d = make(dt, nh, nkv, hs, ps, lens, news, seed=hs + ps, garbage=7.0)
    cap = d["table"].shape[1] * ps
    angle = np.arange(cap)[:, None] * 10000.0 ** (-np.arange(rot // 2) / max(1, rot // 2))
    cos, sin = (torch.from_numpy(f(angle)).float() for f in (np.cos, np.sin))
    check_append(cuda, d, cos, sin, rot, interleaved)


def check_append(cuda, d, cos, sin, rot, interleaved):
    dt, one_each = d["q"].dtype, d["q"].shape[0] == d["lens"].numel() and (d["cu"].diff() == 1).all()
    args = (f64(d["k"]), f64(d["v"]), f64(d["k_cache"]), f64(d["v_cache"]), d["table"].tolist(),
            d["lens"].tolist(), d["cu"].tolist())
    turn = (f64(d["q"]), f64(cos), f64(sin), interleaved) if rot else ()
    q_ref, k_ref, v_ref, written = paged.append(*args, *turn)
    for cu in ([d["cu"], None] if one_each else [d["cu"]]):
        g = to(d, cuda)
        kw = dict(q=g["q"], cos=cos.to(cuda), sin=sin.to(cuda), interleaved=interleaved) if rot else {}
        out = ops.paged_kv_append(g["k"], g["v"], g["k_cache"], g["v_cache"], g["table"], g["lens"],
                                  None if cu is None else cu.to(cuda), **kw)
        # what is not rotated is copied: equal bits; so is every row that was not written
        assert torch.equal(g["v_cache"].cpu(), torch.from_numpy(v_ref).to(dt))
        same = torch.from_numpy(~written)
        assert torch.equal(g["k_cache"].cpu().transpose(1, 2)[same], d["k_cache"].transpose(1, 2)[same])
        if not rot:
            assert out is None
            assert torch.equal(g["k_cache"].cpu(), torch.from_numpy(k_ref).to(dt))
            continue
        # (x c - y s) in FP32: two products and a sum, 3 u (|x| + |y|) with |c|, |s| <= 1, then one
        # rounding to the type; the largest element bounds |x| and |y|
        for a, r in ((out, q_ref), (g["k_cache"], k_ref)):
            tol = 6 * 2.0 ** -24 * 8.0 + np.abs(r) * torch.finfo(dt).eps / 2 + torch.finfo(dt).smallest_normal
            assert np.abs(r).max() <= 8.0 and (np.abs(f64(a) - r) <= tol).all()


def test_append_padding_and_bad_plans(cuda):
    """Rows behind the last sequence, unmapped pages, bad page numbers, lengths beyond the pages and
    negative ones: nothing is stored there, and the rest is."""
    d = make(torch.float32, 4, 2, 64, 8, [20, 9, 24, 12], [6, 4, 8, 5], garbage=7.0)
    for name, h in (("q", 4), ("k", 2), ("v", 2)):          # five rows of padding
        d[name] = torch.cat([d[name], torch.randn(5, h, 64, generator=torch.Generator().manual_seed(1))])
    d["table"][0, 2] = -1
    d["table"][1, 1] = 10 ** 6
    d["lens"][2] = 30                                        # positions 22 .. 29, the pages end at 24
    d["lens"][3] = 3                                         # positions -2 .. 2
    angle = torch.arange(24)[:, None] * 0.1 ** torch.arange(32)
    check_append(cuda, d, angle.cos(), angle.sin(), 64, False)
    d["lens"][:] = torch.tensor([-5, 2 ** 31 - 1, 0, -2 ** 31])
    check_append(cuda, d, angle.cos(), angle.sin(), 64, False)


def test_append_strided(cuda):
    """Tokens that are slices of a packed projection (and misaligned ones), caches that are views of
    (pages, page size, heads, hs) pools or of one pool of both."""
    for dtype in (torch.float32, torch.bfloat16):
        d = make(dtype, 6, 2, 64, 16, [40, 33, 5], [9, 33, 1], garbage=7.0)
        ref = to(d, cuda)
        cos = torch.rand(48, 32, generator=torch.Generator().manual_seed(2)).to(cuda)
        sin = (1 - cos * cos).sqrt()
        want = ops.paged_kv_append(ref["k"], ref["v"], ref["k_cache"], ref["v_cache"], ref["table"],
                                   ref["lens"], ref["cu"], ref["q"], cos, sin)
        g = to(d, cuda)
        for lead in (0, 1):
            packed = torch.cat([g["q"], g["k"], g["v"]], 1).reshape(-1, 640)
            packed = torch.nn.functional.pad(packed, (lead, 24 - lead))[:, lead:lead + 640]
            q, k, v = packed.unflatten(1, (10, 64)).split([6, 2, 2], 1)
            pool = torch.stack([g["k_cache"], g["v_cache"]], 1).transpose(2, 3).contiguous()
            kc, vc = pool[:, 0].transpose(1, 2), pool[:, 1].transpose(1, 2)
            wide = torch.full((3, 7), -1, dtype=torch.int32, device=cuda)
            wide[:, 2:5] = g["table"]
            got = ops.paged_kv_append(k, v, kc, vc, wide[:, 2:5], g["lens"], g["cu"], q, cos, sin)
            assert torch.equal(got, want) and torch.equal(kc, ref["k_cache"])
            assert torch.equal(vc, ref["v_cache"])


# ----------------------------------------------------------------- one new token a sequence
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("hs", [32, 64, 128])
@pytest.mark.parametrize("nh,nkv,ps,lens", [
    (6, 6, 16, [1, 2, 15, 16, 17, 250]),
    (8, 2, 32, [0, 31, 32, 33, 0, 64, 700]),
    (7, 1, 5, [127, 128, 129, 3]),
    (16, 1, 64, [63, 64, 65, 511, 513]),
    (34, 2, 24, [600, 0, 1]),
    (40, 1, 1, [40, 300]),
])
def test_decode(cuda, dtype, hs, nh, nkv, ps, lens):
    check_decode(decode_inputs(dtype, nh, nkv, hs, ps, lens, seed=hs + ps), cuda)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("ps", [16, 12])
def test_decode_long_and_ragged(cuda, dtype, ps):
    """One long sequence among short ones: its positions are split over many workgroups."""
    check_decode(decode_inputs(dtype, 4, 2, 64, ps, [3000, 1, 77, 0, 1500, 16], seed=3), cuda)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("longest", [61, 2300])
def test_decode_many_sequences(cuda, dtype, longest):
    """More sequences than a wave's lanes, short ones only and with long ones among them."""
    lens = [(37 * i) % 61 for i in range(150)]
    lens[7], lens[140] = longest, longest // 2
    check_decode(decode_inputs(dtype, 2, 1, 32, 16, lens, seed=4), cuda)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("ps", [16, 20])
def test_decode_a_workgroup_each(cuda, dtype, ps):
    """As many jobs as the GPU holds workgroups, up to eight tiles each, some empty."""
    longest = 500 if dtype == "float32" else 1000
    lens = [(29 * i) % 41 for i in range(128)]
    lens[3], lens[70], lens[127] = longest, longest // 2 + 1, longest - 129
    check_decode(decode_inputs(dtype, 8, 4, 128, ps, lens, seed=5), cuda)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("ps", [16, 10, 128])
def test_decode_unmapped_pages(cuda, dtype, ps):
    """Holes in the table, whole sequences without a page, bad page numbers, lengths beyond the pages
    and negative ones, and a wider table than any sequence needs."""
    d = decode_inputs(dtype, 6, 2, 64, ps, [500, 300, 40, 2, 90], seed=5, width=60, holes=[(0, 0), (0, 2), (1, 1)])
    d["table"][2, :] = -7
    d["table"][0, 1] = 2 ** 31 - 1
    d["lens"][3] = -3
    check_decode(d, cuda)
    d = decode_inputs(dtype, 6, 2, 64, ps, [4 * ps, 4 * ps], seed=6, width=4)
    d["lens"][0], d["lens"][1] = 4 * ps + 1, 2 ** 31 - 1
    check_decode(d, cuda)


@pytest.mark.parametrize("dtype", ALL)
def test_decode_scores_of_any_size(cuda, dtype):
    """Large scores, masked rows with infinities beside them, a caller's scale (negative too)."""
    d = decode_inputs(dtype, 4, 2, 64, 16, [33, 200], seed=7, scale=6.0, garbage=float("inf"))
    check_decode(d, cuda)
    check_decode(d, cuda, scale=-0.01)
    check_decode(d, cuda, scale=0.0)
    d["q"].fill_(torch.finfo(DTYPES[dtype]).max / 2 if dtype == "float16" else 1e30)
    d["k_cache"].fill_(-1.0)
    O, L = run_decode(d, cuda)              # equal scores of -1e30 and so: the mean of V
    dtp = DTYPES[dtype]
    for b, n in enumerate([33, 200]):
        rows = torch.cat([d["v_cache"][d["table"][b, i]].transpose(0, 1) for i in range(-(-n // 16))])[:n]
        mean = rows.double().mean(0).repeat_interleave(2, 0)
        tol = torch.finfo(dtp).eps / 2 * mean.abs() + rows.double().abs().mean(0).max() * (n * 2.0 ** -23 + 2.0 ** -16)
        assert ((O[b].cpu().double() - mean).abs() <= tol).all()
        assert torch.isfinite(L[b]).all()


def test_decode_infinite_scores(cuda):
    """A key of -inf scores has no weight; a row of only such keys is an empty row."""
    d = decode_inputs("float32", 2, 1, 32, 16, [40, 20], seed=8)
    d["q"] = d["q"].abs() + 0.1
    d["k_cache"][d["table"][0, 1], 0, 3] = -torch.inf
    for i in range(2):
        d["k_cache"][d["table"][1, i]] = -torch.inf
    O, L = run_decode(d, cuda)
    assert torch.isfinite(O).all() and torch.isfinite(L[0]).all()
    assert (O[1] == 0).all() and torch.isneginf(L[1]).all()
    keep = dict(d)
    keep["k_cache"] = d["k_cache"].clone()
    keep["k_cache"][d["table"][0, 1], 0, 3] = -1e30
    assert torch.equal(run_decode(keep, cuda)[0][0], O[0])


@pytest.mark.parametrize("dtype", ALL)
def test_decode_strided(cuda, dtype):
    """Queries of a packed projection and misaligned ones, transposed pools, a table inside a wider
    one: the same bits as the dense call."""
    d = to(decode_inputs(dtype, 6, 2, 64, 16, [100, 7, 33], seed=9, garbage=1.0), cuda)
    want = ops.paged_attention_decode(d["q"], d["k_cache"], d["v_cache"], d["table"], d["lens"])
    pool = torch.stack([d["k_cache"], d["v_cache"]], 1).transpose(2, 3).contiguous()
    kc, vc = pool[:, 0].transpose(1, 2), pool[:, 1].transpose(1, 2)
    wide = torch.full((3, 20), -1, dtype=torch.int32, device=cuda)
    wide[:, 4:4 + d["table"].shape[1]] = d["table"]
    for lead in (0, 1):
        packed = torch.nn.functional.pad(d["q"].reshape(3, -1), (lead, 136 - lead))
        q = packed[:, lead:lead + 384].unflatten(1, (6, 64))
        got = ops.paged_attention_decode(q, kc, vc, wide[:, 4:4 + d["table"].shape[1]], d["lens"])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_large_pool_offsets(cuda, dtype):
    """Pages behind 2^31 elements of the pools, appended to and read."""
    dt, ps, hs = DTYPES[dtype], 64, 128
    pages = (1 << 31) // (ps * hs) + 40
    kc = torch.empty(pages, 1, ps, hs, dtype=dt, device=cuda)
    vc = torch.empty(pages, 1, ps, hs, dtype=dt, device=cuda)
    d = make(dt, 4, 1, hs, ps, [150, 64], [150, 64], seed=11)
    ids = torch.tensor([[pages - 1, pages - 30, pages - 7], [pages - 2, -1, -1]], dtype=torch.int32)
    g = to(d, cuda)
    ops.paged_kv_append(g["k"], g["v"], kc, vc, ids.to(cuda), g["lens"], g["cu"])
    small = dict(d, table=torch.tensor([[39, 10, 33], [38, -1, -1]], dtype=torch.int32),
                 k_cache=kc[pages - 40:].cpu(), v_cache=vc[pages - 40:].cpu())
    big = (kc, vc, ids.to(cuda), g["lens"])
    check_attention(ops.paged_attention_prefill(g["q"], *big, g["cu"]), oracle_attention(small), dt,
                    150, p_round_prefill(dt))
    last = [149, 213]
    q = g["q"][last].contiguous()
    one = dict(small, q=q.cpu())
    check_attention(ops.paged_attention_decode(q, *big),
                    oracle_attention(one, cu=torch.arange(3, dtype=torch.int32)), dt, 150,
                    p_round_decode(dt))


# ----------------------------------------------------------------- packed new tokens
def check_prefill(d, cuda, scale=None):
    g = to(d, cuda)
    got = ops.paged_attention_prefill(g["q"], g["k_cache"], g["v_cache"], g["table"], g["lens"], g["cu"], scale)
    n = max(1, int(d["lens"].clamp(0, d["table"].shape[1] * d["k_cache"].shape[2]).max()))
    check_attention(got, oracle_attention(d, scale), d["q"].dtype, n, p_round_prefill(d["q"].dtype))
    return got


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("hs", [32, 64, 128])
@pytest.mark.parametrize("nh,nkv,ps,lens,news", [
    (2, 2, 16, [1, 2, 65, 130], [1, 2, 65, 130]),
    (4, 1, 64, [200, 63, 0, 64], [33, 63, 0, 1]),
    (6, 2, 5, [150, 9, 77], [20, 9, 77]),
    (7, 1, 24, [100, 31], [37, 31]),
    (20, 1, 128, [300, 40], [13, 2]),
])
def test_prefill(cuda, dtype, hs, nh, nkv, ps, lens, news):
    check_prefill(make(DTYPES[dtype], nh, nkv, hs, ps, lens, news, seed=hs + ps), cuda)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("ps", [16, 12])
def test_prefill_few_rows_long_cache(cuda, dtype, ps):
    check_prefill(make(DTYPES[dtype], 4, 2, 64, ps, [2500, 1700], [5, 3], seed=21), cuda)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("longest", [41, 1500])
def test_prefill_many_sequences(cuda, dtype, longest):
    lens = [(29 * i) % 41 for i in range(100)]
    news = [n // 3 for n in lens]
    lens[70], lens[99] = longest, longest // 2
    check_prefill(make(DTYPES[dtype], 2, 1, 32, 16, lens, news, seed=22), cuda)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("hs,ps", [(32, 16), (64, 40), (128, 64)])
def test_prefill_uneven_tiles(cuda, dtype, hs, ps):
    """Tiles of very different cost, cut anywhere and joined, beside rows of padding, an unmapped page
    and sequences without new tokens."""
    d = make(DTYPES[dtype], 6, 2, hs, ps, [1300, 40, 900, 0, 700, 300], [60, 40, 130, 0, 0, 1], seed=29,
             holes=[(0, 1)])
    d["q"] = torch.cat([d["q"], torch.full((40, 6, hs), torch.nan, dtype=d["q"].dtype)])
    check_prefill(d, cuda)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("hs,ps", [(32, 24), (64, 16), (128, 64)])
def test_prefill_tiles_of_few_parts(cuda, dtype, hs, ps):
    """Whole prompts and continued ones whose tiles two or three workgroups share."""
    lens, news = ([490, 300], [390, 300]) if dtype == "float32" else ([1000, 930], [600, 450])
    d = make(DTYPES[dtype], 4, 2, hs, ps, lens, news, seed=33, holes=[(1, 2)])
    check_prefill(d, cuda)


def test_prefill_fp32_of_any_magnitude_in_parts(cuda):
    """Values beyond the split's range in the middle of a long cache: the parts of the tile that see
    them agree with those that do not."""
    d = make(torch.float32, 4, 2, 64, 16, [1500], [20], seed=30)
    d["v_cache"][d["table"][0, 40]] *= 2.0 ** 110
    d["k_cache"][d["table"][0, 80]] *= 2.0 ** -100
    check_prefill(d, cuda)


def test_plans_of_any_values(cuda):
    """Lengths, pages and row counts that make no sense give some result and touch nothing else."""
    g = torch.Generator().manual_seed(61)
    for dtype in ("float32", "bfloat16"):
        d = to(make(DTYPES[dtype], 4, 2, 64, 16, [700, 40, 900, 33], [40, 40, 20, 3], seed=31, garbage=0.0), cuda)
        guard = torch.full((1 << 20,), 3.0, device=cuda)
        for _ in range(4):
            for name in ("table", "lens", "cu"):
                x = torch.randint(-(2 ** 31), 2 ** 31 - 1, d[name].shape, generator=g, dtype=torch.int64)
                small = torch.randint(-60, 200, d[name].shape, generator=g)
                pick = torch.rand(d[name].shape, generator=g) < 0.5
                d[name].copy_(torch.where(pick, x, small).to(torch.int32))
            c = (d["k_cache"], d["v_cache"], d["table"], d["lens"])
            ops.paged_kv_append(d["k"], d["v"], *c, d["cu"])
            ops.paged_attention_decode(d["q"][:4], *c)
            ops.paged_attention_prefill(d["q"], *c, d["cu"])
            torch.cuda.synchronize()
        assert (guard == 3.0).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("ps", [16, 10])
def test_prefill_padding_and_bad_plans(cuda, dtype, ps):
    """Rows behind the last sequence, holes and bad page numbers, lengths beyond the pages, negative
    ones, and fewer cached tokens than new ones: rows in front of position 0 see nothing."""
    d = make(DTYPES[dtype], 4, 2, 64, ps, [120, 60, 70, 20], [30, 60, 40, 20], seed=23, holes=[(0, 0), (0, 3)])
    d["q"] = torch.cat([d["q"], torch.full((9, 4, 64), torch.nan, dtype=d["q"].dtype)])
    d["table"][1, 0] = -1                                    # its first rows see no key at all
    d["table"][2, 1] = 2 ** 30
    d["lens"][3] = 8
    check_prefill(d, cuda)
    d = make(DTYPES[dtype], 4, 2, 64, ps, [4 * ps, 4 * ps, 30], [20, 7, 9], seed=24, width=4)
    d["lens"][0], d["lens"][1], d["lens"][2] = 4 * ps + 5, 2 ** 31 - 1, -4
    check_prefill(d, cuda)


@pytest.mark.parametrize("dtype", ALL)
def test_prefill_scores_of_any_size(cuda, dtype):
    d = make(DTYPES[dtype], 4, 2, 64, 16, [33, 200], [33, 70], seed=25, scale=6.0, garbage=float("-inf"))
    check_prefill(d, cuda)
    check_prefill(d, cuda, scale=-0.01)


@pytest.mark.parametrize("hs", [32, 64, 128])
@pytest.mark.parametrize("qk,v", [(2.0 ** 60, 1.0), (1.0, 2.0 ** 110), (2.0 ** -70, 2.0 ** -120), (2.0 ** 90, 2.0 ** -60)])
def test_prefill_fp32_of_any_magnitude(cuda, hs, qk, v):
    """Keys and values far from one, beyond the range in which FP32 splits into 16-bit parts; queries
    the other way, so that scores stay ordinary."""
    d = make(torch.float32, 4, 2, hs, 16, [70, 33], [40, 33], seed=27, garbage=0.0)
    d["q"], d["k_cache"], d["v_cache"] = d["q"] / qk, d["k_cache"] * qk, d["v_cache"] * v
    check_prefill(d, cuda)
    d["q"], d["k_cache"] = d["q"] * qk * qk, d["k_cache"] / qk / qk
    check_prefill(d, cuda)


@pytest.mark.parametrize("dtype", ALL)
def test_prefill_infinite_and_huge_scores(cuda, dtype):
    """A key of -inf scores has no weight, rows of only such keys are empty; equal scores of any
    size give the mean of V; a NaN key spoils its sequence alone."""
    dt = DTYPES[dtype]
    d = make(dt, 2, 1, 32, 16, [40, 20], [9, 20], seed=28)
    d["q"] = d["q"].abs() + 0.1
    d["k_cache"][d["table"][0, 1], 0, 3] = -torch.inf
    for i in range(2):
        d["k_cache"][d["table"][1, i]] = -torch.inf
    g = to(d, cuda)
    args = lambda x: (x["q"], x["k_cache"], x["v_cache"], x["table"], x["lens"], x["cu"])  # noqa: E731
    O, L = ops.paged_attention_prefill(*args(g))
    assert torch.isfinite(O).all() and torch.isfinite(L[:9]).all()
    assert (O[9:] == 0).all() and torch.isneginf(L[9:]).all()
    big = torch.finfo(dt).max / 2 if dtype == "float16" else 1e30
    g["q"].fill_(big)
    g["k_cache"].fill_(-1.0)
    O, L = ops.paged_attention_prefill(*args(g))
    rows = torch.cat([d["v_cache"][d["table"][0, i], 0] for i in range(3)]).double()
    for t in range(9):
        n = 40 - 8 + t
        tol = torch.finfo(dt).eps * rows[:n].abs().mean(0).max() + n * 2.0 ** -23
        assert ((O[t].cpu().double() - rows[:n].mean(0)).abs() <= tol).all()
    assert torch.isfinite(L).all()
    g = to(d, cuda)
    g["k_cache"][g["table"][0, 0], 0, 0, 0] = torch.nan
    O, L = ops.paged_attention_prefill(*args(g))
    assert torch.isnan(O[:9]).all() and not torch.isnan(O[9:]).any()


@pytest.mark.parametrize("dtype", ALL)
def test_prefill_strided(cuda, dtype):
    d = to(make(DTYPES[dtype], 6, 2, 64, 16, [100, 7, 33], [40, 7, 30], seed=26, garbage=1.0), cuda)
    want = ops.paged_attention_prefill(d["q"], d["k_cache"], d["v_cache"], d["table"], d["lens"], d["cu"])
    pool = torch.stack([d["k_cache"], d["v_cache"]], 1).transpose(2, 3).contiguous()
    kc, vc = pool[:, 0].transpose(1, 2), pool[:, 1].transpose(1, 2)
    for lead in (0, 1):
        packed = torch.nn.functional.pad(d["q"].reshape(-1, 384), (lead, 136 - lead))
        q = packed[:, lead:lead + 384].unflatten(1, (6, 64))
        got = ops.paged_attention_prefill(q, kc, vc, d["table"], d["lens"], d["cu"])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ----------------------------------------------------------------- together
def test_empty_calls(cuda):
    for dt in DTYPES.values():
        d = to(make(dt, 4, 2, 64, 16, [0, 0], [0, 0]), cuda)
        c = (d["k_cache"], d["v_cache"], d["table"], d["lens"])
        ops.paged_kv_append(d["k"], d["v"], *c, d["cu"])
        O, L = ops.paged_attention_prefill(d["q"], *c, d["cu"])
        assert O.shape == (0, 4, 64) and L.shape == (0, 4)
        O, L = ops.paged_attention_decode(torch.ones(2, 4, 64, dtype=dt, device=cuda), *c)
        assert (O == 0).all() and torch.isneginf(L).all()
        none = torch.empty(0, 3, dtype=torch.int32, device=cuda)
        O, L = ops.paged_attention_decode(d["q"], *c[:2], none, d["lens"][:0])
        assert O.shape == (0, 4, 64)
        O, L = ops.paged_attention_prefill(torch.ones(3, 4, 64, dtype=dt, device=cuda), *c[:2], none,
                                           d["lens"][:0], d["cu"][:1])
        assert (O == 0).all() and torch.isneginf(L).all()
        q = torch.randn(3, 4, 64, device=cuda).to(dt)
        cos = torch.rand(48, 32, device=cuda)
        x = torch.ones(3, 2, 64, dtype=dt, device=cuda)
        assert torch.equal(ops.paged_kv_append(x, x, *c[:2], none, d["lens"][:0], d["cu"][:1], q, cos, cos), q)
        no_pages = torch.empty(2, 0, dtype=torch.int32, device=cuda)
        O, L = ops.paged_attention_decode(torch.ones(2, 4, 64, dtype=dt, device=cuda), *c[:2], no_pages, d["lens"] + 5)
        assert (O == 0).all() and torch.isneginf(L).all()


def rope_tables(n, rot, device):
    angle = torch.arange(n)[:, None] * 10000.0 ** (-torch.arange(rot // 2) * 2 / rot)
    return angle.cos().float().to(device), angle.sin().float().to(device)


@pytest.mark.parametrize("dtype", ALL)
def test_prompt_then_tokens_match_one_pass(cuda, dtype):
    """Prompts through the cache in two chunks and then token by token, rotated on the way: every
    token's attention is that of the whole sequence over itself in float64."""
    dt, nh, nkv, hs, ps = DTYPES[dtype], 6, 2, 64, 16
    total, chunks = [70, 33, 9], [[40, 33, 0], [27, 0, 6]]
    g = torch.Generator().manual_seed(31)
    full = [[torch.randn(n, h, hs, generator=g).to(dt) for h in (nh, nkv, nkv)] for n in total]
    cos, sin = rope_tables(80, hs, cuda)
    table = torch.randperm(15, generator=g).view(3, 5).to(torch.int32).to(cuda)
    kc, vc = (torch.full((15, nkv, ps, hs), torch.nan, dtype=dt, device=cuda) for _ in range(2))
    outs, have, rot_q = [[] for _ in total], [0, 0, 0], [[] for _ in total]

    def step(news, decode):
        rows = [[x[have[b]:have[b] + n] for x in full[b]] for b, n in enumerate(news)]
        q, k, v = (torch.cat([r[i] for r in rows]).to(cuda) for i in range(3))
        for b, n in enumerate(news):
            have[b] += n
        lens = torch.tensor(have, dtype=torch.int32, device=cuda)
        cu = torch.tensor([0] + list(np.cumsum(news)), dtype=torch.int32, device=cuda)
        qr = ops.paged_kv_append(k, v, kc, vc, table, lens, None if decode else cu, q, cos, sin)
        if decode:
            O, L = ops.paged_attention_decode(qr, kc, vc, table, lens)
        else:
            O, L = ops.paged_attention_prefill(qr, kc, vc, table, lens, cu)
        at = 0
        for b, n in enumerate(news):
            outs[b].append((O[at:at + n], L[at:at + n]))
            rot_q[b].append(qr[at:at + n])
            at += n

    for news in chunks:
        step(news, False)
    for _ in range(3):
        step([1 if have[b] < total[b] else 1 for b in range(3)] if all(h < t for h, t in zip(have, total))
             else [int(h < t) for h, t in zip(have, total)], all(h < t for h, t in zip(have, total)))
    for b, n in enumerate(have):
        O, L = (torch.cat([o[i] for o in outs[b]]) for i in range(2))
        d = dict(q=torch.cat(rot_q[b]).cpu(), k_cache=kc.cpu(), v_cache=vc.cpu(), table=table[b:b + 1].cpu(),
                 lens=torch.tensor([n]), cu=torch.tensor([0, n]))
        assert n == total[b]
        check_attention((O, L), oracle_attention(d), dt, n, p_round_prefill(dt))


def test_gpt_generates_through_the_cache(cuda):
    """The small GPT's layers on prompts and then single tokens through the paged cache: the logits of
    its forward on the whole sequences."""
    from cuda_transformer_amd.autograd_fns import CudaLinearLayer
    from cuda_transformer_amd.gpt import GPT, GPTConfig, init_weights_

    cfg = GPTConfig(vocab_size=65, d_model=192, n_heads=3, n_layers=2, block_size=64)
    model = GPT(cfg)
    init_weights_(model, 0, std=0.05)
    model = model.to(cuda)
    B, T, ps, hs = 3, 40, 16, 64
    ids = torch.randint(0, 65, (B, T), generator=torch.Generator().manual_seed(1)).to(cuda)
    with torch.no_grad():
        want, _ = model(ids)
    table = torch.arange(B * 4, dtype=torch.int32).view(B, 4).flip(1).contiguous().to(cuda)
    caches = [[torch.full((B * 4, 3, ps, hs), torch.nan, device=cuda) for _ in range(2)] for _ in model.mha]

    def forward(tokens, start):
        n = tokens.shape[1]
        lens = torch.full((B,), start + n, dtype=torch.int32, device=cuda)
        cu = torch.arange(0, B * n + 1, n, dtype=torch.int32, device=cuda)
        x = model.embedding.embedding(tokens) + model.embedding.positional.weight[start:start + n]
        for block, (kc, vc) in zip(model.mha, caches):
            qkv = CudaLinearLayer.apply(block.ln1(x), block.attn.qkv_weight, block.attn.qkv_bias)
            q, k, v = (t.unflatten(-1, (3, hs)) for t in qkv.view(B * n, -1).chunk(3, -1))
            ops.paged_kv_append(k, v, kc, vc, table, lens, cu)
            att = (ops.paged_attention_decode(q, kc, vc, table, lens) if n == 1 else
                   ops.paged_attention_prefill(q, kc, vc, table, lens, cu))[0]
            x = x + CudaLinearLayer.apply(att.view(B, n, -1), block.attn.out_weight, block.attn.out_bias)
            x = x + block.mlp(block.ln2(x))
        return CudaLinearLayer.apply(model.ln(x), model.lm_head_weights, model.lm_head_bias)

    with torch.no_grad():
        got = [forward(ids[:, :30], 0)] + [forward(ids[:, i:i + 1], i) for i in range(30, T)]
    # the same FP32 operations up to attention's order of sums: the suite's bar for FP32 attention
    torch.testing.assert_close(torch.cat(got, 1), want, rtol=1e-4, atol=1e-5)


def test_two_graphs_and_streams(cuda):
    """A serving step captured twice, replayed on two streams with eager work between: every replay
    equals the eager step bit for bit."""
    def state(seed):
        return to(make(torch.bfloat16, 8, 2, 128, 16, [900, 30, 0, 2000], [1, 1, 1, 1], seed=seed, width=130), cuda)

    def step(d):
        cos, sin = d["cos"], d["sin"]
        q = ops.paged_kv_append(d["k"], d["v"], d["k_cache"], d["v_cache"], d["table"], d["lens"], None, d["q"], cos, sin)
        one = ops.paged_attention_decode(q, d["k_cache"], d["v_cache"], d["table"], d["lens"])
        many = ops.paged_attention_prefill(q, d["k_cache"], d["v_cache"], d["table"], d["lens"], d["cu"])
        return (q, *one, *many)

    states = [state(41), state(42)]
    for d in states:
        d["cos"], d["sin"] = rope_tables(130 * 16, 128, cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for d in states:
            step(d)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for d in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(d))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        for i, d in enumerate(states):
            d["q"].copy_(torch.randn(d["q"].shape, generator=torch.Generator().manual_seed(100 + 10 * rep + i)))
            d["lens"].copy_(torch.tensor([900 - 7 * rep, 30 + rep, i, 2000 - rep]))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for d, got in zip(states, outs):
            got = [t.clone() for t in got]
            for a, b in zip(got, step(d)):
                assert torch.equal(a, b), f"replay {rep}"


def test_shared_prefix_pages(cuda):
    """Two sequences that share their first pages: each reads them as its own."""
    d = decode_inputs("bfloat16", 4, 2, 64, 16, [70, 70], seed=51)
    d["table"][1, :3] = d["table"][0, :3]
    check_decode(d, cuda)
