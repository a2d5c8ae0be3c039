"""The serving operators on the GPU: attention over packed prompts, appending to the 8-bit cache, single-token attention over
it, each against a plain implementation in 64 bits, and a run of the three together.

Tolerances. Attention: with u the half step of the storage type and A = sum_j p_j |v_j|, the output is off by at most
u |o| (its own rounding) + w A, where w covers the rounding of a probability to 16 bits on its way into the matrix product
(u of that type; nothing where probabilities stay in fp32), the 2^x of the kernels (below 7.5e-5) and the fp32 scores
(D products: below 1e-4 of a nat for the sizes here). A probability that is rounded to f16 is stored times 2^7 relative to a
running maximum m that the true one does not fall short of: the spacing of f16 is 2^-24 below 2^-14, so that a probability far
below the largest is off by at most 2^-25 * 2^-7 = 2^-32 of 2^m, and the output by at most 2^-32 sum_j |v_j| (the sum that
divides it is at least 2^m). Codes and scales of the 8-bit cache have to be equal."""
import numpy as np
import pytest
import torch

import vknn_b200
from vknn_b200 import capi

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"e4m3": torch.float8_e4m3fn, "i8": torch.int8}
SMALL = 2e-4  # 2^x and scores


def half_step(dt):
    return torch.finfo(dt).eps / 2


def offsets(lengths, device="cuda"):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device=device)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def attention64(q, k, v, scale, causal):
    """q [nq,Hq,D], k/v [nk,Hkv,D] in float64: o and the two sums of its bound, NaN rows where nothing is visible."""
    group = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    x = torch.einsum("qhd,khd->hqk", q, k) * scale
    if causal:
        hidden = torch.arange(k.shape[0], device=q.device) > torch.arange(q.shape[0], device=q.device)[:, None] + (k.shape[0] - q.shape[0])
        x = x.masked_fill(hidden, -torch.inf)
    p = torch.softmax(x, -1) if k.shape[0] else x
    seen = torch.isfinite(p).all(-1).T[..., None] if k.shape[0] else torch.zeros(q.shape[0], q.shape[1], 1, dtype=torch.bool, device=q.device)
    o, a = (torch.einsum("hqk,khd->qhd", torch.nan_to_num(p), t) for t in (v, v.abs()))
    nan = torch.full_like(o, torch.nan)
    if not k.shape[0]:
        return nan, nan
    vsum = torch.einsum("hqk,khd->qhd", torch.isfinite(x).to(v.dtype), torch.nan_to_num(v.abs()))
    return torch.where(seen, o, nan), torch.where(seen, torch.stack([a, 2.0 ** -32 * vsum]), nan)


def check(got, ref, sums, dt, p_dt, what=""):
    """sums: (sum_j p_j |v_j|, 2^-32 sum_j |v_j|)."""
    a, far = sums if sums.dim() > ref.dim() else (sums, torch.zeros_like(sums))
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), (what, "NaN in other places", int(torch.isnan(got).sum()), int(torch.isnan(ref).sum()))
    off = torch.nan_to_num((got - ref).abs())
    w = (half_step(p_dt) if p_dt is not None else 0.0) + SMALL
    tol = torch.nan_to_num(half_step(dt) * ref.abs() + w * a + (far if p_dt == torch.float16 else 0.0)) + (6e-8 if dt == torch.float16 else 1e-30)
    assert bool((off <= tol).all()), (what, "largest excess", float((off / tol.clamp(min=1e-30)).max()))


# ---- attention over packed sequences --------------------------------------------------------------------------------

IMPLS = [(vknn_b200.IMPL_SIMT, "simt"), (vknn_b200.IMPL_AUTO, "auto")]


@pytest.fixture(params=[i for i, _ in IMPLS], ids=[n for _, n in IMPLS])
def impl_ctx(ctx, request):
    ctx.set_impl(request.param)
    yield ctx
    ctx.set_impl(vknn_b200.IMPL_AUTO)


def packed_case(seed, lq, lk, hq, hkv, d, dt):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = randn(g, sum(lq), hq, d).to(dt)
    k, v = (randn(g, sum(lk), hkv, d).to(dt) for _ in range(2))
    return q, k, v


def check_packed(ctx, q, k, v, lq, lk, causal, scale, what=""):
    dt = q.dtype
    o = torch.full(q.shape, 7.0, dtype=dt, device="cuda")
    ctx.attn_prefill_packed(q, k, v, o, scale, offsets(lq), cu_k=offsets(lk), causal=causal)
    ctx.sync()
    aq = ak = 0
    for nq, nk in zip(lq, lk):
        ref, a = attention64(q[aq:aq + nq].double(), k[ak:ak + nk].double(), v[ak:ak + nk].double(), scale, causal)
        check(o[aq:aq + nq], ref, a, dt, dt if dt != torch.float32 else None, (what, nq, nk))
        aq, ak = aq + nq, ak + nk
    return o


LENGTHS = {"one": ([1], [1]), "edges": ([5, 0, 1, 127, 128, 129, 256, 257], None), "tiny": ([1, 1, 2, 3, 1, 0, 0, 1], None), "long": ([700, 31, 1100], None),
           "prefix": ([1, 7, 130, 0, 300], [400, 7, 131, 5, 555]), "hidden": ([9, 40, 300, 4], [3, 0, 140, 4])}


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (6, 2, 128)])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_packed_lengths(impl_ctx, dt, hq, hkv, d, lengths, causal):
    lq, lk = LENGTHS[lengths]
    lk = lk or lq
    q, k, v = packed_case(1, lq, lk, hq, hkv, d, DT[dt])
    check_packed(impl_ctx, q, k, v, lq, lk, causal, d ** -0.5)


@pytest.mark.parametrize("d", [8, 40, 96, 256])
@pytest.mark.parametrize("dt", ["f32", "f16"])
def test_packed_other_head_sizes_and_fp32(ctx, dt, d):
    lq, lk = [33, 0, 9], [40, 3, 9]
    q, k, v = packed_case(2, lq, lk, 4, 2, d, DT[dt])
    check_packed(ctx, q, k, v, lq, lk, True, d ** -0.5)


def test_packed_many_random_batches(ctx):
    r = np.random.default_rng(5)
    for n in range(12):
        nseq, d, hkv, group = int(r.integers(1, 20)), int(r.choice([64, 128])), int(r.choice([1, 2, 3])), int(r.choice([1, 2, 5]))
        lq = [int(x) for x in r.integers(0, int(r.choice([4, 150, 600])), nseq)]
        lk = [x + int(r.integers(0, 300)) for x in lq] if n % 2 else lq
        if not sum(lq):
            continue
        q, k, v = packed_case(n, lq, lk, hkv * group, hkv, d, torch.bfloat16 if n % 3 else torch.float16)
        check_packed(ctx, q, k, v, lq, lk, bool(n % 4), d ** -0.5, n)


def test_packed_views_of_one_projection(impl_ctx):
    lq, hq, hkv, d = [50, 200, 3], 6, 2, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = randn(g, sum(lq), hq + 2 * hkv, d).half()
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    out = torch.zeros(sum(lq), 2 * hq, d, dtype=torch.float16, device="cuda")
    impl_ctx.attn_prefill_packed(q, k, v, out[:, ::2], d ** -0.5, offsets(lq))  # (heads every second place)
    dense = torch.zeros(sum(lq), hq, d, dtype=torch.float16, device="cuda")
    impl_ctx.attn_prefill_packed(q.contiguous(), k.contiguous(), v.contiguous(), dense, d ** -0.5, offsets(lq))
    impl_ctx.sync()
    assert torch.equal(out[:, ::2], dense) and not out[:, 1::2].any()


def test_packed_unaligned_strides(ctx):
    """Bases and strides that a 16-byte load cannot follow."""
    lq, h, d = [20, 41], 2, 64
    g = torch.Generator(device="cuda").manual_seed(4)
    wide = randn(g, 3, sum(lq), h, d + 3).half()
    q, k, v = (wide[i, :, :, 1:d + 1] for i in range(3))
    check_packed(ctx, q, k, v, lq, lq, True, d ** -0.5)


def test_packed_rows_outside_the_sequences_stay(impl_ctx):
    h, d = 2, 128
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k, v = (randn(g, 400, h, d).half() for _ in range(3))
    o = torch.full((400, h, d), 3.0, dtype=torch.float16, device="cuda")
    cu = torch.tensor([10, 140, 140, 301], dtype=torch.int32, device="cuda")
    impl_ctx.attn_prefill_packed(q, k, v, o, d ** -0.5, cu)
    impl_ctx.sync()
    assert bool((o[:10] == 3).all()) and bool((o[301:] == 3).all())
    for a, b in ((10, 140), (140, 301)):
        ref, m = attention64(q[a:b].double(), k[a:b].double(), v[a:b].double(), d ** -0.5, True)
        check(o[a:b], ref, m, torch.float16, torch.float16)


def test_packed_offsets_outside_the_tensor_are_clamped(impl_ctx):
    h, d = 2, 64
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k, v = (randn(g, 100, h, d).half() for _ in range(3))
    o, want = (torch.zeros(100, h, d, dtype=torch.float16, device="cuda") for _ in range(2))
    impl_ctx.attn_prefill_packed(q, k, v, o, d ** -0.5, torch.tensor([-5, 40, 1000000], dtype=torch.int32, device="cuda"))
    impl_ctx.attn_prefill_packed(q, k, v, want, d ** -0.5, torch.tensor([0, 40, 100], dtype=torch.int32, device="cuda"))
    impl_ctx.sync()
    assert torch.equal(o, want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("d", [64, 128])
def test_packed_neighbours_do_not_leak(impl_ctx, d, bad):
    """The sequences before and behind hold nothing but infinities or NaN; a hidden key's K may be anything too."""
    lq, h = [3, 129, 70, 1, 250, 6], 2
    q, k, v = packed_case(8, lq, lq, h, h, d, torch.bfloat16)
    at = np.concatenate([[0], np.cumsum(lq)])
    for i in (0, 2, 5):
        for t in (q, k, v):
            t[at[i]:at[i + 1]] = bad
    o = torch.zeros_like(q)
    impl_ctx.attn_prefill_packed(q, k, v, o, d ** -0.5, offsets(lq))
    impl_ctx.sync()
    for i in (1, 3, 4):
        s = slice(at[i], at[i + 1])
        ref, a = attention64(q[s].double(), k[s].double(), v[s].double(), d ** -0.5, True)
        check(o[s], ref, a, torch.bfloat16, torch.bfloat16, i)


def test_packed_maximum_grows_late(impl_ctx):
    """Scores that rise along the keys: the running maximum moves in every tile."""
    lq, h, d = [600, 300], 2, 64
    q, k, v = packed_case(9, lq, lq, h, h, d, torch.float16)
    k *= torch.linspace(0.1, 6.0, sum(lq), device="cuda")[:, None, None]
    k = k.half()
    check_packed(impl_ctx, q, k, v, lq, lq, True, d ** -0.5)
    check_packed(impl_ctx, q, k, v, lq, lq, False, d ** -0.5)


def test_packed_same_bits_again_on_another_stream_and_in_a_graph(ctx):
    lq, hq, hkv, d = [513, 40, 0, 300], 8, 2, 128
    q, k, v = packed_case(10, lq, lq, hq, hkv, d, torch.bfloat16)
    cu, want = offsets(lq), torch.zeros_like(q)
    ctx.attn_prefill_packed(q, k, v, want, d ** -0.5, cu)
    other, o = torch.cuda.Stream(), torch.zeros_like(q)
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        ctx.attn_prefill_packed(q, k, v, o, d ** -0.5, cu)
    other.synchronize()
    assert torch.equal(o, want)
    graph, o2 = torch.cuda.CUDAGraph(), torch.zeros_like(q)
    with torch.cuda.graph(graph):
        ctx.attn_prefill_packed(q, k, v, o2, d ** -0.5, cu)
    for n in ([100, 400, 53, 300], lq):  # other lengths of the same total, without a new capture
        cu.copy_(offsets(n))
        graph.replay()
        torch.cuda.synchronize()
        o.zero_()
        ctx.attn_prefill_packed(q, k, v, o, d ** -0.5, offsets(n))
        torch.cuda.synchronize()
        assert torch.equal(o2, o)
    assert torch.equal(o2, want)


def test_packed_output_strides_that_16_bytes_cannot_follow(ctx):
    lq, hq, hkv, d = [150, 3, 260], 4, 2, 64
    q, k, v = packed_case(11, lq, lq, hq, hkv, d, torch.float16)
    o = torch.full((sum(lq), hq, d + 3), 5.0, dtype=torch.float16, device="cuda")
    want = torch.zeros_like(q)
    ctx.attn_prefill_packed(q, k, v, o[:, :, 1:d + 1], d ** -0.5, offsets(lq))
    ctx.attn_prefill_packed(q, k, v, want, d ** -0.5, offsets(lq))
    ctx.sync()
    assert torch.equal(o[:, :, 1:d + 1], want) and bool((o[:, :, 0] == 5).all()) and bool((o[:, :, d + 1:] == 5).all())


def check_like_simt(ctx, lq, lk, hq, hkv, d, causal=True):
    """Against the SIMT kernel, which the tests above compare with 64 bits: each is within its own bound of the exact value, so they
    differ by the sum of the two."""
    q, k, v = packed_case(12, lq, lk, hq, hkv, d, torch.bfloat16)
    o, want, a = torch.full_like(q, 9.0), torch.full_like(q, 9.0), torch.zeros_like(q)
    cu_q, cu_k = offsets(lq), offsets(lk)
    ctx.attn_prefill_packed(q, k, v, o, d ** -0.5, cu_q, cu_k, causal)
    ctx.set_impl(vknn_b200.IMPL_SIMT)
    ctx.attn_prefill_packed(q, k, v, want, d ** -0.5, cu_q, cu_k, causal)
    ctx.attn_prefill_packed(q, k, v.abs(), a, d ** -0.5, cu_q, cu_k, causal)  # sum p |v|
    ctx.set_impl(vknn_b200.IMPL_AUTO)
    ctx.sync()
    assert torch.equal(torch.isnan(o), torch.isnan(want))  # rows without a key
    u = half_step(torch.bfloat16)
    o, w, s = (torch.nan_to_num(x.double()) for x in (o, want, a))
    s = s * (1 + 2 * u)  # (a is itself rounded)
    tol = 2 * u * w.abs() * (1 + u) + (u + 2 * SMALL) * s * (1 + u)
    assert bool(((o - w).abs() <= tol).all())


@pytest.mark.parametrize("hq,hkv,d,nseq,hi", [(32, 8, 128, 300, 60), (20, 20, 64, 300, 60), (18, 6, 128, 280, 70), (4, 2, 64, 900, 5), (6, 6, 128, 700, 6), (64, 2, 64, 40, 300)],
                         ids=["pairs_many_rounds", "rows_many_rounds", "odd_group", "more_units_than_are_ranked", "rows_more_units", "wide_group"])
def test_packed_many_sequences(ctx, hq, hkv, d, nseq, hi):
    """Many rounds per CTA, more units than one CTA ranks, groups of odd and of large size."""
    lq = [int(x) for x in np.random.default_rng(nseq).integers(0, hi + 1, nseq)]
    check_like_simt(ctx, lq, lq, hq, hkv, d)


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "full"])
@pytest.mark.parametrize("hq,hkv,d,nseq,hi,some", [(64, 2, 64, 130, 60, 20), (32, 8, 128, 700, 6, 50), (6, 6, 128, 700, 6, 50), (6, 6, 64, 700, 200, 50)],
                         ids=["ranked", "pairs", "rows", "rows64"])
def test_packed_long_runs_of_sequences_without_keys(ctx, hq, hkv, d, nseq, hi, some, causal):
    """Keys for the first sequences and (beyond what is ranked) the last; dozens of rounds of a CTA in between have nothing to compute."""
    lq = [int(x) for x in np.random.default_rng(nseq).integers(1, hi + 1, nseq)]
    lk = [n + 3 if i < some or i >= nseq - some // 2 else 0 for i, n in enumerate(lq)]
    check_like_simt(ctx, lq, lk, hq, hkv, d, causal)
    check_like_simt(ctx, lq, [0] * (nseq - 1) + [5], hq, hkv, d, causal)
    check_like_simt(ctx, lq, [5] + [0] * (nseq - 1), hq, hkv, d, causal)


@pytest.mark.parametrize("nseq,hi", [(120, 90), (700, 20)], ids=["ranked", "unranked"])
def test_packed_many_sequences_replayed_with_other_offsets(ctx, nseq, hi):
    hq, hkv, d, r = 32, 8, 64, np.random.default_rng(6)
    first = [int(x) for x in r.integers(0, hi + 1, nseq)]
    total = sum(first)
    q, k, v = packed_case(14, first, first, hq, hkv, d, torch.float16)
    cu, o, want = offsets(first), torch.zeros_like(q), torch.zeros_like(q)
    ctx.attn_prefill_packed(q, k, v, o, d ** -0.5, cu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.attn_prefill_packed(q, k, v, o, d ** -0.5, cu)
    far = 2.0 ** -32 * float(v.double().abs().sum(0).max())
    cuts = [sorted(int(x) for x in r.integers(0, total + 1, nseq - 1)) for _ in range(2)] + [[total] * (nseq - 1), [0] * (nseq - 1)]
    for cut in cuts:
        cu.copy_(torch.tensor([0] + cut + [total], dtype=torch.int32))
        graph.replay()
        ctx.attn_prefill_packed(q, k, v, want, d ** -0.5, cu)  # launched, not replayed
        torch.cuda.synchronize()
        assert torch.equal(o, want)
        ctx.set_impl(vknn_b200.IMPL_SIMT)
        a = torch.zeros_like(q)
        ctx.attn_prefill_packed(q, k, v, want, d ** -0.5, cu)
        ctx.attn_prefill_packed(q, k, v.abs(), a, d ** -0.5, cu)
        ctx.set_impl(vknn_b200.IMPL_AUTO)
        ctx.sync()
        # both within half a step of fp16 and of P in fp16 of the exact value, which loses 2^-32 |v| per key where P is subnormal
        u = half_step(torch.float16)
        w, s = want.double(), a.double() * (1 + 2 * u)
        assert bool(((o.double() - w).abs() <= 2 * u * w.abs() * (1 + u) + (u + 2 * SMALL) * s * (1 + u) + 1.2e-7 + far).all())


def test_packed_a_sequence_of_more_units_than_are_ranked(ctx):
    check_like_simt(ctx, [66000, 40], [66000, 40], 2, 1, 64)
    check_like_simt(ctx, [40, 33100, 1], [50, 33100, 900], 2, 2, 128)


def test_packed_keys_shared_by_a_broadcast_stride(ctx):
    """One kv head expanded over all of them, and one value row for all tokens (strides of 0): the same as the copies."""
    lq, h, d = [60, 131], 4, 64
    q, k, v = packed_case(15, lq, lq, h, 1, d, torch.float16)
    ke, ve = k.expand(-1, h, -1), v[:1].expand(sum(lq), h, d).contiguous()[:, :1].expand(-1, h, -1)
    o, want = torch.zeros_like(q), torch.zeros_like(q)
    ctx.attn_prefill_packed(q, ke, ve, o, d ** -0.5, offsets(lq))
    ctx.attn_prefill_packed(q, ke.contiguous(), ve.contiguous(), want, d ** -0.5, offsets(lq))
    ctx.sync()
    ref, a = attention64(q[:60].double(), ke[:60].double(), ve[:60].double(), d ** -0.5, True)
    check(o[:60], ref, a, torch.float16, torch.float16)
    check(want[:60], ref, a, torch.float16, torch.float16)


def test_packed_same_offsets_for_queries_and_a_longer_key_buffer(ctx):
    """cu_k may be the very tensor cu_q while K and V have more rows than Q."""
    lq, h, d = [30, 41], 2, 64
    q, _, _ = packed_case(13, lq, lq, h, h, d, torch.float16)
    _, k, v = packed_case(14, lq, [300], h, h, d, torch.float16)
    cu, o, want = offsets(lq), torch.zeros_like(q), torch.zeros_like(q)
    ctx.attn_prefill_packed(q, k, v, o, d ** -0.5, cu, cu_k=cu)
    ctx.attn_prefill_packed(q, k[:71], v[:71], want, d ** -0.5, cu)
    ctx.sync()
    assert torch.equal(o, want)


def test_packed_nothing_to_do(ctx):
    e = torch.zeros(0, 2, 64, dtype=torch.float16, device="cuda")
    ctx.attn_prefill_packed(e, e, e, e, 1.0, offsets([0, 0]))
    q = torch.ones(3, 2, 64, dtype=torch.float16, device="cuda")
    o = torch.zeros_like(q)
    ctx.attn_prefill_packed(q, e, e, o, 1.0, offsets([3]), cu_k=offsets([0]))
    ctx.sync()
    assert bool(torch.isnan(o).all())


# ---- the 8-bit cache -------------------------------------------------------------------------------------------------

class Cache:
    def __init__(self, b, hkv, lmax, d, block, codes, fill=None):
        self.block, self.codes = block, CODES[codes]
        self.k, self.v = (torch.zeros(b, hkv, lmax, d, dtype=self.codes, device="cuda") for _ in range(2))
        self.ks, self.vs = (torch.zeros(b, hkv, lmax // block, device="cuda") for _ in range(2))
        if fill is not None:  # bits nobody may look at
            for t in (self.k, self.v):
                t.view(torch.uint8).fill_(fill)
            for t in (self.ks, self.vs):
                t.fill_(float("nan"))

    @property
    def args(self):
        return self.k, self.v, self.ks, self.vs

    def clone(self):
        c = object.__new__(Cache)
        c.block, c.codes = self.block, self.codes
        c.k, c.v, c.ks, c.vs = (t.clone() for t in self.args)
        return c

    def same(self, other):
        return all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(self.args, other.args))


def scale64(top, codes):
    if not np.isfinite(top):
        return np.float32(np.nan)
    if top == 0:
        return np.float32(0)
    if codes == torch.int8:
        return max(np.float32(top) / np.float32(127), np.float32(2.0 ** -126))
    e = -126
    while top > 448.0 * 2.0 ** e:
        e += 1
    return np.float32(2.0 ** e)


def encode64(x, s, codes):
    """x float64 array -> code bytes."""
    y = x / np.float64(s) if s > 0 else np.zeros_like(x)
    if codes == torch.int8:
        return np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8)
    return torch.from_numpy(y.astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def append64(cache, x, which, lens, cu):
    """The definition, block by block, on the host: changes the cache's codes and scales of K or V."""
    codes, scales = (cache.k, cache.ks) if which == "k" else (cache.v, cache.vs)
    c, s, x = codes.cpu(), scales.cpu().numpy().copy(), x.double().cpu().numpy()
    raw, block, lmax = c.view(torch.uint8).numpy(), cache.block, c.shape[2]
    for b, start in enumerate(lens):
        n = cu[b + 1] - cu[b]
        end = min(start + n, lmax)
        if start < 0 or start >= lmax:
            continue
        for blk in range(start // block, -(-end // block)) if n else ():
            lo = max(start, blk * block)
            hi = min(end, (blk + 1) * block)
            for h in range(c.shape[1]):
                new = x[cu[b] + lo - start:cu[b] + hi - start, h]
                scale = scale64(np.abs(new).max(), cache.codes)
                if lo > blk * block:
                    was = s[b, h, blk]
                    scale = np.float32(np.nan) if np.isnan(was) or np.isnan(scale) else max(was, scale)
                    if scale > was:
                        old = c[b, h, blk * block:lo].double().numpy() * np.float64(was)
                        raw[b, h, blk * block:lo] = encode64(old, scale, cache.codes)
                raw[b, h, lo:hi] = encode64(new, scale, cache.codes)
                s[b, h, blk] = scale
    codes.copy_(c)
    scales.copy_(torch.from_numpy(s))


def append_both(ctx, cache, k, v, lens, cu=None):
    """Appends through the library and through the definition; both have to leave the same bits. Returns the cache."""
    want = cache.clone()
    at = cu if cu is not None else list(range(len(lens) + 1))
    ctx.kv_append_q8(k, v, *cache.args, torch.tensor(lens, dtype=torch.int32, device="cuda"),
                     cu=torch.tensor(cu, dtype=torch.int32, device="cuda") if cu is not None else None)
    ctx.sync()
    append64(want, k, "k", lens, at)
    append64(want, v, "v", lens, at)
    for name, a, b in zip(("k", "v", "k_scale", "v_scale"), cache.args, want.args):
        if name.endswith("scale"):
            assert torch.equal(torch.nan_to_num(a, nan=-1.0), torch.nan_to_num(b, nan=-1.0)), name
        else:
            d = a.view(torch.uint8) != b.view(torch.uint8)
            assert not d.any(), (name, int(d.sum()), d.nonzero()[:4].tolist())
    return cache


def rows(seed, t, hkv, d, dt, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(randn(g, t, hkv, d) * torch.exp(spread * randn(g, t, 1, 1))).to(dt) for _ in range(2)]


@pytest.mark.parametrize("codes", ["e4m3", "i8"])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("d,block", [(64, 32), (128, 64), (256, 128), (128, 32), (64, 128)])
def test_append_prompts_then_tokens(ctx, dt, d, block, codes):
    lens = [0, 1, block - 1, block, block + 5, 2 * block]
    new = [3, 2 * block, 1, 0, 2 * block + 7, block + 1]
    cu = [int(x) for x in np.concatenate([[0], np.cumsum(new)])]
    cache = Cache(len(lens), 2, 6 * block, d, block, codes)
    k, v = rows(1, max(lens) * len(lens), 2, d, DT[dt])
    append_both(ctx, cache, k, v, [0] * len(lens), [int(x) for x in np.concatenate([[0], np.cumsum(lens)])])
    k, v = rows(2, cu[-1] + 3, 2, d, DT[dt])  # (rows behind the last sequence belong to nobody)
    append_both(ctx, cache, k, v, lens, cu)
    held = [a + b for a, b in zip(lens, new)]
    for step in range(3):
        k, v = rows(10 + step, len(lens), 2, d, DT[dt])
        append_both(ctx, cache, k, v, held)
        held = [x + 1 for x in held]


@pytest.mark.parametrize("codes", ["e4m3", "i8"])
def test_append_tokens_whose_scale_grows(ctx, codes):
    """One token at a time, each larger than those before it: the older codes are requantised again and again."""
    cache = Cache(3, 2, 64, 64, 32, codes)
    for step in range(40):
        k, v = rows(step, 3, 2, 64, torch.bfloat16)
        append_both(ctx, cache, k * 1.17 ** step, v * 1.9 ** step, [step, step, step])


@pytest.mark.parametrize("codes", ["e4m3", "i8"])
def test_append_values_on_the_border_between_codes(ctx, codes):
    """Quotients that lie exactly in the middle between two codes, or a step of their type beside it."""
    d, block = 64, 32
    scale = 2.0 ** -3
    mid = (torch.arange(-127, 127, device="cuda").float() + 0.5) if codes == "i8" else torch.tensor(
        [17.0, 19, 21, 23, 25, 1.0625, 1.1875, 0.0009765625, 0.0029296875, 27, 34, 38, 232, 248, 432, 0.0205078125], device="cuda").repeat(16)[:254]
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        x = torch.zeros(2, block, d, device="cuda")
        x[0, :4].view(-1)[:254] = mid * scale
        x[0, 4:8].view(-1)[:254] = torch.nextafter(mid * scale, torch.zeros_like(mid))
        x[0, 8:12].view(-1)[:254] = torch.nextafter(mid * scale, torch.full_like(mid, 1e9))
        x[0, 12:, 0] = (127 if codes == "i8" else 448) * scale
        x[1] = x[0] * 0.7313  # a scale that is not a power of two
        k = x.to(dt).transpose(0, 1)
        append_both(ctx, Cache(1, 2, 64, d, block, codes), k, -k, [0], [0, block])


@pytest.mark.parametrize("codes", ["e4m3", "i8"])
def test_append_zeros_tiny_and_huge(ctx, codes):
    cache = Cache(5, 1, 64, 64, 32, codes)
    for step, sizes in enumerate([(0.0, 1e-39, 1e-30, 3e38, 1.0), (1e-38, 1e-45, 0.0, 1.0, 3e38), (0.0, 0.0, 1e-20, 1e30, 1e-38)]):
        k, v = rows(step, 5, 1, 64, torch.float32, spread=0.0)
        k = k.clamp(-1, 1) * torch.tensor(sizes, device="cuda")[:, None, None]
        append_both(ctx, cache, k, -k, [step] * 5)


@pytest.mark.parametrize("codes", ["e4m3", "i8"])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_append_infinities_and_nan_mark_their_block(ctx, codes, bad):
    cache = Cache(2, 2, 96, 64, 32, codes)
    k, v = rows(1, 80, 2, 64, torch.float16)
    k[37, 1, 5] = bad
    append_both(ctx, cache, k, v, [0, 3], [0, 50, 80])
    assert bool(torch.isnan(cache.ks[0, 1, 1])) and int(torch.isnan(cache.ks).sum()) == 1 and int(torch.isnan(cache.vs).sum()) == 0
    k, v = rows(2, 2, 2, 64, torch.float16)
    append_both(ctx, cache, k, v, [50, 33])  # behind it in the same block: stays marked
    assert int(torch.isnan(cache.ks).sum()) == 1


def test_append_onto_scales_of_the_callers_own(ctx):
    """Scales this library would not have chosen (not a power of two, larger than needed, smaller)."""
    for codes in ("e4m3", "i8"):
        cache = Cache(4, 2, 64, 128, 32, codes)
        k, v = rows(3, 40, 2, 128, torch.bfloat16)
        append_both(ctx, cache, k, v, [0] * 4, [0, 10, 20, 30, 40])
        for s in (cache.ks, cache.vs):
            s *= torch.tensor([0.3, 1.37, 5.0, 0.011], device="cuda")[:, None, None]
        k, v = rows(4, 4, 2, 128, torch.bfloat16)
        append_both(ctx, cache, k, v, [10] * 4)


def nearest_e4m3(x, s):
    """The e4m3 code nearest to x / s, ties to even, by exact comparisons: x is compared with (middle between two codes) * s, of at
    most 5 + 24 bits, in float64. x: float64 of at most 28 bits, s: float32, broadcast."""
    values = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()  # codes 0 to 126, ascending
    mids = (values[1:] + values[:-1]) / 2
    a, s = np.broadcast_arrays(np.abs(x), np.asarray(s, dtype=np.float64))
    code = np.zeros(a.shape, dtype=np.uint8)
    for c, mid in enumerate(mids):  # from code c on to c + 1
        code += ((a > mid * s) | ((a == mid * s) & (c % 2 == 1))).astype(np.uint8)
    return code | (np.signbit(x).astype(np.uint8) << 7)


def test_append_e4m3_rounds_once_with_any_scale(ctx):
    """Scales that are not powers of two: quotients so close to the middle between two codes that they round to it in fp32."""
    r, hkv, b, d, block = np.random.default_rng(17), 64, 4, 64, 32
    # new rows beside a token whose block has such a scale
    s = (2.0 ** r.integers(-20, 20, (b, hkv)) * r.uniform(1.0, 2.0, (b, hkv))).astype(np.float32)
    mid = np.array([17, 19, 21, 23, 25, 27, 29, 31, 1.0625, 1.1875, 3.25, 5.75, 0.4375 + 1 / 64, 3 * 2.0 ** -10, 2.0 ** -10, 5 * 2.0 ** -10], dtype=np.float64)
    x = (mid * s[..., None].astype(np.float64)).astype(np.float32)
    x = np.concatenate([x, np.nextafter(x, np.float32(0)), np.nextafter(x, np.float32(np.inf)), -x], -1)  # [b, hkv, 64]
    cache = Cache(b, hkv, block, d, block, "e4m3")
    cache.ks.copy_(torch.from_numpy(s)[..., None])
    cache.vs.copy_(torch.from_numpy(s)[..., None])
    k, one = torch.from_numpy(x).cuda(), torch.ones(b, dtype=torch.int32, device="cuda")
    ctx.kv_append_q8(k, -k, *cache.args, one)
    ctx.sync()
    for t, y in ((cache.k, x), (cache.v, -x)):
        got, want = t[:, :, 1].view(torch.uint8).cpu().numpy(), nearest_e4m3(y.astype(np.float64), s[..., None])
        assert np.array_equal(got, want), int((got != want).sum())
    assert np.array_equal(cache.ks[..., 0].cpu().numpy(), s)
    # older codes whose scale grows to a power of two
    v = 1 + np.arange(1, 8, dtype=np.float64) / 8
    pairs = [(m, c) for m in mid[:8] / 16 for c in v if m < c][: b * hkv]
    s = np.array([np.float32(m / c) for m, c in pairs], dtype=np.float32)
    s = np.concatenate([s, np.nextafter(s, np.float32(0)), np.nextafter(s, np.float32(1))])
    s = np.resize(s, (b, hkv))
    held = np.resize(np.concatenate([np.arange(0x20, 0x50), 0x80 + np.arange(0x30, 0x40)]), d).astype(np.uint8)
    cache = Cache(b, hkv, block, d, block, "e4m3")
    for t, z in ((cache.k, cache.ks), (cache.v, cache.vs)):
        t.view(torch.uint8)[:, :, 0] = torch.from_numpy(held).cuda()
        z.copy_(torch.from_numpy(s)[..., None])
    k = torch.full((b, hkv, d), 300.0, device="cuda")  # asks for the scale 1
    ctx.kv_append_q8(k, k, *cache.args, one)
    ctx.sync()
    assert bool((cache.ks == 1).all()) and bool((cache.vs == 1).all())
    value = torch.from_numpy(held).view(torch.float8_e4m3fn).double().numpy()
    want = nearest_e4m3(value * s[..., None].astype(np.float64), np.float32(1))
    for t in (cache.k, cache.v):
        got = t[:, :, 0].view(torch.uint8).cpu().numpy()
        assert np.array_equal(got, want), int((got != want).sum())


def test_append_rows_that_do_not_fit_and_idle_sequences(ctx):
    cache = Cache(5, 2, 64, 64, 32, "e4m3")
    k, v = rows(5, 5, 2, 64, torch.float16)
    append_both(ctx, cache, k, v, [63, 64, -1, 1000, 0])
    k, v = rows(6, 50, 2, 64, torch.float16)
    append_both(ctx, cache, k, v, [60, -3, 64, 31, 50], [0, 10, 20, 30, 40, 50])


@pytest.mark.parametrize("codes", ["e4m3", "i8"])
def test_append_strided_and_unaligned_rows(ctx, codes):
    hkv, d = 3, 64
    g = torch.Generator(device="cuda").manual_seed(7)
    qkv = randn(g, 40, 4 + 2 * hkv, d).half()
    append_both(ctx, Cache(2, hkv, 64, d, 32, codes), qkv[:, 4:4 + hkv], qkv[:, 4 + hkv:], [0, 5], [0, 33, 40])
    odd = randn(g, 2, 40, hkv, d + 1).half()
    append_both(ctx, Cache(2, hkv, 64, d, 32, codes), odd[0, :, :, 1:], odd[1, :, :, :d], [0, 5], [0, 33, 40])


def test_append_twice_and_in_a_graph(ctx):
    """Appending the same rows again changes nothing; a captured append follows kv_len."""
    cache = Cache(3, 2, 128, 128, 64, "i8")
    k, v = rows(8, 3, 2, 128, torch.bfloat16)
    append_both(ctx, cache, k, v, [0, 10, 64])
    again = cache.clone()
    ctx.kv_append_q8(k, v, *again.args, torch.tensor([0, 10, 64], dtype=torch.int32, device="cuda"))
    ctx.sync()
    assert again.same(cache)
    lens, graph = torch.tensor([1, 11, 65], dtype=torch.int32, device="cuda"), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.kv_append_q8(k, v, *cache.args, lens)
    want = cache.clone()
    for step in range(3):
        nk, nv = rows(20 + step, 3, 2, 128, torch.bfloat16)
        k.copy_(nk)
        v.copy_(nv)
        append64(want, nk, "k", lens.tolist(), [0, 1, 2, 3])
        append64(want, nv, "v", lens.tolist(), [0, 1, 2, 3])
        graph.replay()
        lens += 1
    torch.cuda.synchronize()
    assert cache.same(want)


# ---- attention over the 8-bit cache -----------------------------------------------------------------------------------

def filled(seed, b, hkv, lmax, d, block, codes):
    """A cache of random codes and scales (K and V as large as in use), no call of the library."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = Cache(b, hkv, lmax, d, block, codes)
    for t, s in ((c.k, c.ks), (c.v, c.vs)):
        w = randn(g, *t.shape)
        if codes == "i8":
            t.copy_((w * 40).round().clamp(-127, 127))
            s.copy_(0.025 * torch.exp(0.5 * randn(g, *s.shape)))
        else:
            t.view(torch.uint8).copy_((w * 64).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8))
            s.copy_(torch.exp2(torch.randint(-8, -4, s.shape, generator=g, device="cuda").float()))
    return c


def decode64(q, cache, lens, scale):
    refs, sums = [], []
    for i, n in enumerate(lens):
        n = max(0, min(n, cache.k.shape[2]))
        k, v = (t[i, :, :n].double() * s[i].double().repeat_interleave(cache.block, 1)[:, :n, None] for t, s in ((cache.k, cache.ks), (cache.v, cache.vs)))
        r, a = attention64(q[i:i + 1].double(), k.transpose(0, 1), v.transpose(0, 1), scale, False)
        refs.append(r)
        sums.append(a if a.dim() > r.dim() else torch.stack([a, a]))
    return torch.cat(refs), torch.cat(sums, 1)


def check_decode(ctx, q, cache, lens, scale, what=""):
    o = torch.full_like(q, 5.0)
    ctx.attn_decode_q8(q, *cache.args, o, scale, kv_len=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    ctx.sync()
    ref, a = decode64(q, cache, lens, scale)
    check(o, ref, a, q.dtype, torch.float16, what)
    return o


def queries(seed, b, hq, d, dt):
    return randn(torch.Generator(device="cuda").manual_seed(seed), b, hq, d).to(DT[dt])


@pytest.mark.parametrize("codes", ["e4m3", "i8"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 8, 12, 16, 17])
@pytest.mark.parametrize("d,block", [(64, 32), (128, 64), (256, 128)])
def test_decode_q8_shapes(impl_ctx, d, block, group, dt, codes):
    lens = [1, 0, 31, 32, 33, block, 300, 511, 512, 4 * block - 1]
    cache = filled(1, len(lens), 2, 512, d, block, codes)
    check_decode(impl_ctx, queries(2, len(lens), 2 * group, d, dt), cache, lens, d ** -0.5)


@pytest.mark.parametrize("codes", ["e4m3", "i8"])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("group", [1, 3, 8, 12, 16])
@pytest.mark.parametrize("d,block", [(64, 32), (128, 64), (256, 128)])
def test_decode_q8_shapes_of_a_longer_cache(ctx, d, block, group, dt, codes):
    """The same with room for so many keys that the work is split over the keys."""
    lens = [1, 0, 31, 32, 33, block, 300, 1407, 1408, 4 * block - 1]
    cache = filled(1, len(lens), 2, 1408, d, block, codes)
    check_decode(ctx, queries(2, len(lens), 2 * group, d, dt), cache, lens, d ** -0.5)


@pytest.mark.parametrize("codes", ["e4m3", "i8"])
@pytest.mark.parametrize("hq,d,block,dt", [(17, 64, 32, "bf16"), (32, 128, 64, "f16"), (71, 256, 128, "bf16")])
def test_decode_q8_large_groups_over_a_long_cache(ctx, hq, d, block, dt, codes):
    """More than 16 query heads on one kv head: the SIMT form, here with thousands of keys for every warp to walk."""
    lens = [9001, 0, 1, 8192]
    cache = filled(41, len(lens), 1, 9216, d, block, codes)
    check_decode(ctx, queries(42, len(lens), hq, d, dt), cache, lens, d ** -0.5)


@pytest.mark.parametrize("room", [768, 1024, 1280])
@pytest.mark.parametrize("hkv", [1, 37, 38, 74, 75, 148, 149])
def test_decode_q8_around_the_number_of_multiprocessors(ctx, hkv, room):
    """Where the choice between a block of threads per kv head and equal shares changes; the first tokens of a cache of any room."""
    for d, block, b in ((64, 32, 2), (128, 128, 4), (256, 64, 1)):
        for lmax in (room, room // 2):
            lens = [lmax, lmax // 3, 0, 1][:b]
            check_decode(ctx, queries(23, b, hkv, d, "bf16"), filled(22, b, hkv, lmax, d, block, "e4m3"), lens, d ** -0.5, (d, lmax))


@pytest.mark.parametrize("codes,fill", [("e4m3", 0x7f), ("i8", 0x80)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_q8_never_uses_what_lies_behind_in_a_longer_cache(ctx, codes, fill, d):
    lens, block = [1, 33, 90, 1290, 0, 2048], 64
    cache = filled(24, 6, 2, 2048, d, block, codes)
    for i, n in enumerate(lens):
        for t in (cache.k, cache.v):
            t.view(torch.uint8)[i, :, n:] = fill
        for s in (cache.ks, cache.vs):
            s[i, :, -(-n // block):] = float("nan")
    q = queries(25, 6, 4, d, "f16")
    o = torch.zeros_like(q)
    ctx.attn_decode_q8(q, *cache.args, o, d ** -0.5, kv_len=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    ctx.sync()
    ref, a = decode64(q, cache, lens, d ** -0.5)
    check(o, ref, a, torch.float16, torch.float16)
    cache.ks[0, 1, 0] = float("nan")  # a marked block in use
    cache.vs[3, 0, 20] = float("nan")
    ctx.attn_decode_q8(q, *cache.args, o, d ** -0.5, kv_len=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    ctx.sync()
    bad = torch.isnan(o).all(-1)
    assert bad.tolist() == [[False, False, True, True], [False] * 4, [False] * 4, [True, True, False, False], [True] * 4, [False] * 4]
    assert int(torch.isnan(o).any(-1).sum()) == int(bad.sum())


@pytest.mark.parametrize("codes", ["e4m3", "i8"])
@pytest.mark.parametrize("b,hq,hkv,lmax,lens", [
    (1, 8, 1, 16384, [16001]), (1, 12, 12, 512, [331]), (3, 16, 8, 4096, [4096, 1, 2500]), (40, 4, 2, 2048, None), (2, 8, 2, 32768, [32768, 70]), (70, 8, 8, 128, None)],
    ids=["one_long", "one_short", "uneven", "batch", "long_and_short", "many_short"])
def test_decode_q8_lengths(ctx, b, hq, hkv, lmax, lens, codes):
    lens = lens or [int(x) for x in np.random.default_rng(3).integers(0, lmax + 1, b)]
    for dt, d, block in (("f16", 128, 64), ("bf16", 64, 32)):
        check_decode(ctx, queries(4, b, hq, d, dt), filled(5, b, hkv, lmax, d, block, codes), lens, d ** -0.5)


def test_decode_q8_random_batches(ctx):
    r = np.random.default_rng(11)
    for n in range(16):
        b, hkv, group, d = int(r.integers(1, 30)), int(r.choice([1, 2, 5])), int(r.integers(1, 17)), int(r.choice([64, 128, 256]))
        block = int(r.choice([32, 64, 128]))
        lmax = block * int(r.integers(1, 2600 // block))
        lens = [int(x) for x in r.integers(-2, lmax + 3, b)] if n % 2 else [int(lmax * x ** 4) for x in r.random(b)]
        check_decode(ctx, queries(n, b, hkv * group, d, "bf16" if n % 3 else "f16"), filled(n, b, hkv, lmax, d, block, "i8" if n % 2 else "e4m3"), lens, d ** -0.5, n)


@pytest.mark.parametrize("codes,fill", [("e4m3", 0x7f), ("e4m3", 0xff), ("i8", 0x80)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_q8_never_uses_what_lies_behind(impl_ctx, codes, fill, d):
    """NaN codes and NaN scales behind the last token, in its own block and in the following ones."""
    lens, block = [1, 33, 90, 128, 0], 32
    cache, clean = filled(6, 5, 2, 160, d, block, codes), None
    for i, n in enumerate(lens):
        for t in (cache.k, cache.v):
            t.view(torch.uint8)[i, :, n:] = fill
        for s in (cache.ks, cache.vs):
            s[i, :, -(-n // block):] = float("nan")
    q = queries(7, 5, 4, d, "f16")
    o = torch.zeros_like(q)
    impl_ctx.attn_decode_q8(q, *cache.args, o, d ** -0.5, kv_len=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    impl_ctx.sync()
    ref, a = decode64(q, cache, lens, d ** -0.5)
    check(o, ref, a, torch.float16, torch.float16)


def test_decode_q8_marked_block_answers_nan(impl_ctx):
    cache = filled(8, 3, 2, 256, 64, 32, "e4m3")
    cache.ks[0, 1, 2] = float("nan")
    cache.vs[2, 0, 0] = float("nan")
    q = queries(9, 3, 4, 64, "f16")
    o = torch.zeros_like(q)
    impl_ctx.attn_decode_q8(q, *cache.args, o, 0.125, kv_len=torch.tensor([200, 200, 7], dtype=torch.int32, device="cuda"))
    impl_ctx.sync()
    bad = torch.isnan(o).all(-1)
    assert bad.tolist() == [[False, False, True, True], [False] * 4, [True, True, False, False]] and int(torch.isnan(o).any(-1).sum()) == int(bad.sum())


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_decode_q8_scales_and_queries_of_any_size(impl_ctx, dt):
    """Block scales that differ by many powers of two, zero scales, and queries near the ends of their type."""
    cache = filled(10, 4, 2, 512, 128, 64, "e4m3")
    g = torch.Generator(device="cuda").manual_seed(1)
    cache.vs *= torch.exp2(torch.randint(-20, 20, cache.vs.shape, generator=g, device="cuda").float())
    cache.vs[1] *= 2.0 ** -60
    cache.ks[2, :, 1] = 0
    cache.vs[2, :, 0] = 0
    q = queries(11, 4, 8, 128, dt)
    q[3] *= 2e-5 if dt == "f16" else 1e-25
    q[0, :, ::2] = 0
    check_decode(impl_ctx, q, cache, [512, 511, 130, 400], 0.05)
    if dt == "bf16":  # beyond the range of fp16, brought back by the scale
        check_decode(impl_ctx, (q * 1e20).to(torch.bfloat16), cache, [512, 511, 130, 400], 0.05e-20)
    big = filled(12, 4, 2, 512, 128, 64, "e4m3")
    check_decode(impl_ctx, q, big, [512, 511, 130, 400], -0.05)  # a negative scale


def test_decode_q8_maximum_grows_late(impl_ctx):
    cache = filled(13, 2, 1, 2048, 64, 32, "i8")
    cache.ks *= torch.linspace(0.05, 4.0, 64, device="cuda")
    check_decode(impl_ctx, queries(14, 2, 4, 64, "f16"), cache, [2048, 1999], 0.125)


@pytest.mark.parametrize("lmax", [4096, 768])  # (lengths beyond the cache count as its length)
def test_decode_q8_same_bits_again_with_a_workspace_on_a_stream_and_in_a_graph(ctx, lmax):
    b, hq, hkv, d, block = 5, 8, 2, 128, 64
    cache, q = filled(15, b, hkv, lmax, d, block, "e4m3"), queries(16, b, hq, d, "bf16")
    lens = torch.tensor([4096, 1, 0, 3000, 777], dtype=torch.int32, device="cuda")
    want = torch.zeros_like(q)
    ctx.attn_decode_q8(q, *cache.args, want, d ** -0.5, kv_len=lens)
    need = ctx.attn_decode_q8_workspace_bytes(b, hq, hkv, lmax, d)
    ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")  # whatever it held before
    outs = [torch.zeros_like(q) for _ in range(3)]
    ctx.attn_decode_q8(q, *cache.args, outs[0], d ** -0.5, kv_len=lens, workspace=ws)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        ctx.attn_decode_q8(q, *cache.args, outs[1], d ** -0.5, kv_len=lens)
    other.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    got = [torch.zeros_like(q) for _ in range(2)]
    spaces = [torch.zeros(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for gr, o, w in zip(graphs, got, spaces):
        with torch.cuda.graph(gr):
            ctx.attn_decode_q8(q, *cache.args, o, d ** -0.5, kv_len=lens, workspace=w)
    for _ in range(3):
        for gr in graphs:
            gr.replay()
    torch.cuda.synchronize()
    for o in outs[:2] + got:
        assert torch.equal(torch.nan_to_num(o, nan=9.0), torch.nan_to_num(want, nan=9.0))
    lens.copy_(torch.tensor([5, 4096, 100, 0, 4000], dtype=torch.int32, device="cuda"))  # other lengths, same graph
    graphs[0].replay()
    torch.cuda.synchronize()
    ref, a = decode64(q, cache, lens.tolist(), d ** -0.5)
    check(got[0], ref, a, torch.bfloat16, torch.float16)


def test_decode_q8_more_sequences_than_one_launch_holds(ctx):
    b, hq, hkv, lmax, d, block = 1500, 4, 2, 128, 64, 32
    lens = [int(x) for x in np.random.default_rng(9).integers(0, lmax + 1, b)]
    cache, q = filled(17, b, hkv, lmax, d, block, "i8"), queries(18, b, hq, d, "bf16")
    check_decode(ctx, q, cache, lens, d ** -0.5)


def test_decode_q8_captured_without_a_workspace():
    """The context's own scratch does not grow during a capture: a clean error, nothing launched, and the context goes on working.
    After one ordinary call of the shape the same capture is fine; short caches need no scratch at all."""
    fresh = vknn_b200.Context(0)
    try:
        hq, hkv, d, block, lens = 8, 2, 128, 64, torch.tensor([4000, 77, 300], dtype=torch.int32, device="cuda")
        cache, short, q = filled(31, 3, hkv, 4096, d, block, "e4m3"), filled(32, 3, hkv, 256, d, block, "e4m3"), queries(33, 3, hq, d, "f16")
        want, o = torch.zeros_like(q), torch.full_like(q, 5.0)
        attend = lambda c, out, **kw: fresh.attn_decode_q8(q, *c.args, out, d ** -0.5, kv_len=lens, **kw)  # noqa: E731
        attend(short, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attend(short, o)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want)
        n0, graph, mark = fresh.launch_count(), torch.cuda.CUDAGraph(), torch.zeros(1, device="cuda")
        with torch.cuda.graph(graph):
            mark += 1
            with pytest.raises(vknn_b200.VkcError) as e:
                attend(cache, o)
        assert e.value.code == -1 and fresh.launch_count() == n0
        attend(cache, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attend(cache, o)
        graph.replay()
        fresh.sync()
        torch.cuda.synchronize()
        assert torch.equal(o, want)
        ref, a = decode64(q, cache, lens.tolist(), d ** -0.5)
        check(o, ref, a, torch.float16, torch.float16)
        # with a workspace a context that has none of its own captures at once
        other = vknn_b200.Context(0)
        try:
            ws, graph = torch.empty(other.attn_decode_q8_workspace_bytes(3, hq, hkv, 4096, d), dtype=torch.uint8, device="cuda"), torch.cuda.CUDAGraph()
            o.zero_()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                other.attn_decode_q8(q, *cache.args, o, d ** -0.5, kv_len=lens, workspace=ws)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want)
        finally:
            other.close()
    finally:
        fresh.close()


@pytest.mark.parametrize("lmax", [4096, 1024])
def test_decode_q8_two_calls_at_once(ctx, lmax):
    """Two streams, a workspace each; and one after the other on two streams with the context's own scratch."""
    d, block = 128, 64
    cases = [(filled(19 + i, 3, 2, lmax, d, block, "e4m3"), queries(21 + i, 3, 8, d, "f16"), torch.tensor([4000 - 900 * i, 77, 3000], dtype=torch.int32, device="cuda")) for i in range(2)]
    want = []
    for c, q, lens in cases:
        o = torch.zeros_like(q)
        ctx.attn_decode_q8(q, *c.args, o, d ** -0.5, kv_len=lens)
        ctx.sync()
        want.append(o)
    need, streams = ctx.attn_decode_q8_workspace_bytes(3, 8, 2, lmax, d), [torch.cuda.Stream() for _ in range(2)]
    spaces = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for own in (True, False):
        got = [[torch.zeros_like(q) for _ in range(4)] for _, q, _ in cases]
        torch.cuda.synchronize()
        for n in range(4):
            for i, (c, q, lens) in enumerate(cases):
                with torch.cuda.stream(streams[i]):
                    ctx.attn_decode_q8(q, *c.args, got[i][n], d ** -0.5, kv_len=lens, workspace=spaces[i] if own else None)
        torch.cuda.synchronize()
        for i in range(2):
            for o in got[i]:
                assert torch.equal(o, want[i]), (own, i)


def test_cache_beyond_32_bit_offsets(ctx):
    """Rows of a cache whose codes lie more than 2^32 bytes behind its first. Keys and values are zero but for the last block of each
    sequence, so that the exact answer is a short sum: the zero keys have score 0 and weigh (length - block) together."""
    b, hkv, hq, d, block, lmax = 2, 1, 4, 128, 128, (1 << 25) + 256
    k, v = (torch.zeros(b, hkv, lmax, d, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(b, hkv, lmax // block, device="cuda") for _ in range(2))
    assert k[1].data_ptr() - k.data_ptr() > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(23)
    n, start = 100, lmax - block
    new = [(randn(g, b * n, hkv, d) * 2).to(torch.bfloat16) for _ in range(2)]
    held = torch.tensor([start, start], dtype=torch.int32, device="cuda")
    ctx.kv_append_q8(*new, k, v, ks, vs, held, cu=offsets([n, n]))
    held += n
    q, o = (randn(g, b, hq, d) * 3).to(torch.float16), torch.zeros(b, hq, d, dtype=torch.float16, device="cuda")
    ctx.attn_decode_q8(q, k, v, ks, vs, o, 0.3, kv_len=held)
    ctx.sync()
    for i in range(b):
        kk, vv = (t[i, 0, start:start + n].double() * s[i, 0, -1].double() for t, s in ((k, ks), (v, vs)))
        assert float((kk - new[0][i * n:(i + 1) * n, 0].double()).abs().max()) <= 2.0 ** -4 * float(kk.abs().max())
        x = q[i].double() @ kk.T * 0.3
        top = x.amax(-1, keepdim=True).clamp(min=0)
        p = torch.exp(x - top)
        p = p / (p.sum(-1, keepdim=True) + start * torch.exp(-top))
        check(o[i], p @ vv, torch.stack([p @ vv.abs(), 2.0 ** -32 * vv.abs().sum(0).expand(hq, -1)]), torch.float16, torch.float16)
    del k, v


# ---- the three together ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("codes", ["e4m3", "i8"])
def test_prompts_then_tokens_as_a_server_runs_them(ctx, codes):
    """Prompts of different lengths through packed attention, their keys and values into the 8-bit cache, then tokens one by
    one. Every attention is compared with 64 bits over what the cache holds, and what it holds with the values stored:
    a code is off by at most half a step (int8: scale / 2 plus the requantisations; e4m3: 2^-4 of the value or the
    smallest step)."""
    hq, hkv, d, block, lmax, dt = 8, 2, 128, 32, 192, torch.bfloat16
    prompt = [70, 1, 0, 129]
    g = torch.Generator(device="cuda").manual_seed(21)
    qkv = randn(g, sum(prompt), hq + 2 * hkv, d).to(dt)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    cu, cache = offsets(prompt), Cache(4, hkv, lmax, d, block, codes, fill=0x7f)
    held = torch.zeros(4, dtype=torch.int32, device="cuda")
    o = torch.zeros(sum(prompt), hq, d, dtype=dt, device="cuda")
    ctx.attn_prefill_packed(q, k, v, o, d ** -0.5, cu)
    ctx.kv_append_q8(k, v, *cache.args, held, cu=cu)
    held += cu[1:] - cu[:-1]
    history = [[k[cu[i]:cu[i + 1]].clone(), v[cu[i]:cu[i + 1]].clone()] for i in range(4)]
    for step in range(5):
        tq, tk, tv = randn(g, 4, hq, d).to(dt), randn(g, 4, hkv, d).to(dt), randn(g, 4, hkv, d).to(dt)
        ctx.kv_append_q8(tk, tv, *cache.args, held)
        held += 1
        out = torch.zeros_like(tq)
        ctx.attn_decode_q8(tq, *cache.args, out, d ** -0.5, kv_len=held)
        ctx.sync()
        lens = held.tolist()
        ref, a = decode64(tq, cache, lens, d ** -0.5)
        check(out, ref, a, dt, torch.float16, step)
        for i in range(4):
            history[i] = [torch.cat([h, t[i:i + 1]]) for h, t in zip(history[i], (tk, tv))]
            for t, s, h in zip((cache.k, cache.v), (cache.ks, cache.vs), history[i]):
                per = s[i].double().repeat_interleave(block, 1)[:, :lens[i], None]
                off = (t[i, :, :lens[i]].double() * per - h.double().transpose(0, 1)).abs()
                x = h.double().transpose(0, 1).abs()
                # a code written once is off by half a step; each of at most `step + 1` growths of the scale adds at most half a step of its own
                tol = per * 0.5 * (step + 2) if codes == "i8" else x * 2.0 ** -4 + per * 2.0 ** -10 * (step + 2)
                assert bool((off <= tol * (1 + 1e-6)).all()), (i, step)
    for i in range(4):
        s = slice(int(cu[i]), int(cu[i + 1]))
        ref, a = attention64(q[s].double(), k[s].double(), v[s].double(), d ** -0.5, True)
        check(o[s], ref, a, dt, dt)


@pytest.mark.parametrize("lmax", [256, 4096])
@pytest.mark.parametrize("codes", ["e4m3", "i8"])
def test_steps_behind_the_product_that_writes_their_rows(ctx, codes, lmax):
    """Projection, append and attention of several steps one right behind the other, over the same buffers: each kernel may start while
    the one before it still runs, and has to see what that one wrote. The same bits as with a wait after every call."""
    b, hq, hkv, d, block, dt, steps, width = 6, 8, 2, 128, 32, torch.bfloat16, 12, 512
    g = torch.Generator(device="cuda").manual_seed(51)
    x, w = (randn(g, *s).to(dt) * 0.2 for s in ((steps, b, width), (width, (hq + 2 * hkv) * d)))
    lens = [torch.tensor([1, 31, 100, 0, 5, 64], dtype=torch.int32, device="cuda") + s for s in range(steps + 1)]
    ws = torch.zeros(ctx.attn_decode_q8_workspace_bytes(b, hq, hkv, lmax, d), dtype=torch.uint8, device="cuda")
    start, qkv = filled(52, b, hkv, lmax, d, block, codes), torch.zeros(b, (hq + 2 * hkv) * d, dtype=dt, device="cuda")
    q, out = torch.zeros(b, hq, d, dtype=dt, device="cuda"), torch.zeros(steps, b, hq, d, dtype=dt, device="cuda")

    def run(cache, between):
        for s in range(steps):
            ctx.gemm(x[s], w, qkv)
            between()
            rows3 = qkv.view(b, hq + 2 * hkv, d)
            ctx.kv_append_q8(rows3[:, hq:hq + hkv], rows3[:, hq + hkv:], *cache.args, lens[s])
            between()
            ctx.gemm(x[s], wq, q.view(b, hq * d))
            between()
            ctx.attn_decode_q8(q, *cache.args, out[s], d ** -0.5, kv_len=lens[s + 1], workspace=ws)
            between()

    idle, wq = lambda: None, w[:, :hq * d].contiguous()
    cache = start.clone()
    run(cache, torch.cuda.synchronize)
    want, kept = out.clone(), cache.clone()
    graph, cache = torch.cuda.CUDAGraph(), start.clone()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        run(cache, idle)
    for _ in range(5):
        for t, s in zip(cache.args, start.args):
            t.copy_(s)
        out.zero_()
        qkv.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and cache.same(kept)
        for t, s in zip(cache.args, start.args):
            t.copy_(s)
        out.zero_()
        run(cache, idle)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and cache.same(kept)
    assert bool(torch.isfinite(want).all())


# ---- refusals -----------------------------------------------------------------------------------------------------------

def test_refusals_of_the_serving_operators(ctx):
    n0 = ctx.launch_count()
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    cache = Cache(2, 2, 64, 64, 32, "e4m3")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    q, kv = z(6, 4, 64), z(6, 2, 64)
    for call in (lambda: ctx.attn_prefill_packed(q, kv, kv, q, 1.0, lens.long()), lambda: ctx.attn_prefill_packed(q, kv, kv[:5], q, 1.0, lens),
                 lambda: ctx.attn_prefill_packed(q, kv.float(), kv, q, 1.0, lens), lambda: ctx.attn_prefill_packed(q, kv, kv, q, 1.0, lens, cu_k=lens[:1]),
                 lambda: ctx.attn_prefill_packed(q.cpu(), kv, kv, q, 1.0, lens), lambda: ctx.attn_prefill_packed(q.transpose(0, 2), kv, kv, q, 1.0, lens),
                 lambda: ctx.kv_append_q8(kv, kv, cache.k, cache.v, cache.ks[..., :1], cache.vs, lens), lambda: ctx.kv_append_q8(q, q, *cache.args, lens),
                 lambda: ctx.kv_append_q8(kv, kv, *cache.args, lens.float()), lambda: ctx.kv_append_q8(kv, kv, *cache.args, lens[:1]),
                 lambda: ctx.kv_append_q8(kv, kv, z(2, 2, 64, 64), z(2, 2, 64, 64), cache.ks, cache.vs, lens),
                 lambda: ctx.attn_decode_q8(z(3, 4, 64), *cache.args, z(3, 4, 64), 1.0, lens), lambda: ctx.attn_decode_q8(z(2, 4, 64), *cache.args, z(2, 4, 64).bfloat16(), 1.0, lens),
                 lambda: ctx.attn_decode_q8(z(2, 4, 64), cache.k[:, :, ::2], cache.v[:, :, ::2], cache.ks, cache.vs, z(2, 4, 64), 1.0, lens)):
        with pytest.raises(ValueError):
            call()
    for code, call in (
            (-1, lambda: ctx.attn_prefill_packed(z(6, 3, 64), kv, kv, z(6, 3, 64), 1.0, lens)), (-1, lambda: ctx.attn_prefill_packed(q, z(7, 2, 64), z(7, 2, 64), q, 1.0, lens)),
            (-1, lambda: ctx.attn_prefill_packed(z(6, 4, 264), z(6, 2, 264), z(6, 2, 264), z(6, 4, 264), 1.0, lens)),
            (-1, lambda: ctx.kv_append_q8(kv, kv, *cache.args, lens)),  # six rows for two sequences without cu
            (-2, lambda: ctx.kv_append_q8(kv[:2], kv[:2], cache.k, cache.v, z(2, 2, 1, dt=torch.float32).repeat(1, 1, 4), z(2, 2, 4, dt=torch.float32), lens)),  # block of 16
            (-2, lambda: ctx.kv_append_q8(z(2, 2, 32), z(2, 2, 32), z(2, 2, 64, 32, dt=torch.int8), z(2, 2, 64, 32, dt=torch.int8), cache.ks, cache.vs, lens)),
            (-1, lambda: ctx.attn_decode_q8(z(2, 5, 64), *cache.args, z(2, 5, 64), 1.0, lens)),
            (-2, lambda: ctx.attn_decode_q8(z(2, 4, 64, dt=torch.float32), *cache.args, z(2, 4, 64, dt=torch.float32), 1.0, lens)),
            (-1, lambda: ctx.attn_decode_q8(z(2, 4, 64), *cache.args, z(2, 4, 64), 1.0, lens, workspace=z(1, dt=torch.uint8)))):
        with pytest.raises(vknn_b200.VkcError) as e:
            call()
        assert e.value.code == code
    assert ctx.launch_count() == n0


def test_outputs_that_share_memory_are_refused(ctx):
    """Rows of O under one another's address: whichever is stored last would stay."""
    q, kv = (torch.zeros(*s, dtype=torch.float16, device="cuda") for s in ((6, 4, 64), (6, 2, 64)))
    cu, n0 = torch.tensor([0, 2, 6], dtype=torch.int32, device="cuda"), ctx.launch_count()
    for o in (q[:, :1].expand(6, 4, 64), q[:1].expand(6, 4, 64)):
        with pytest.raises(vknn_b200.VkcError) as e:
            ctx.attn_prefill_packed(q, kv, kv, o, 1.0, cu)
        assert e.value.code == -1 and "share memory" in str(e.value)
    assert ctx.launch_count() == n0
    one = torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda")  # a single token: its stride is of no account
    ctx.attn_prefill_packed(one, one, one, torch.zeros_like(one).as_strided((1, 4, 64), (0, 64, 1)), 1.0, torch.tensor([0, 1], dtype=torch.int32, device="cuda"))
    ctx.sync()


def test_misaligned_pointers_are_refused(ctx):
    """C callers only: a tensor cannot lie at such an address. Nothing is launched."""
    n0, lib = ctx.launch_count(), ctx.lib
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    q, kv, lens, cache = z(2, 4, 64), z(2, 2, 64), z(3, dt=torch.int32), Cache(2, 2, 64, 64, 32, "e4m3")
    p, codes, scales, n = q.data_ptr(), [t.data_ptr() for t in (cache.k, cache.v)], [t.data_ptr() for t in (cache.ks, cache.vs)], lens.data_ptr()
    kvp = [kv.data_ptr()] * 2
    calls = [(lib.vkc_attn_prefill_packed, capi.PACKED_ARGS, [p, *kvp, p, 2, 4, 2, 64, 2, 2, n, n, *[0] * 8, 1.0, 1, vknn_b200.F16], (0, 1, 2, 3, 10, 11)),
             (lib.vkc_kv_append_q8, capi.APPEND_ARGS, [*kvp, *codes, *scales, 2, 2, 64, 64, 32, 2, n, n, *[0] * 4, vknn_b200.F16, vknn_b200.E4M3], (0, 1, 2, 3, 4, 5, 12, 13)),
             (lib.vkc_attn_decode_q8, capi.DECODE_Q8_ARGS, [p, *codes, *scales, p, 2, 4, 2, 64, 64, 32, n, 0, 0, 1.0, vknn_b200.F16, vknn_b200.E4M3], (0, 1, 2, 3, 4, 5, 12))]
    for f, struct, args, pointers in calls:
        for i in pointers:
            bad = list(args)
            bad[i] += 1
            assert f(ctx.h, struct.pack(*bad), 1) == -1, (f, i)
            assert b"aligned" in lib.vkc_last_error(ctx.h)
    assert ctx.launch_count() == n0
