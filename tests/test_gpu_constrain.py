"""GPU tests of cdclq.tune's constraints on logits, against their definition in 64 bits.

Tolerances. In f32 a quotient or product by repetition, the product frequency * c, its sum with presence, the
subtraction and the addition of the bias (a sum of n values: n - 1 roundings) are off by 2^-24 of their values each; the
result is rounded once to its type (u). All magnitudes on the way are below |l| rep + |freq c| + |pres| + sum |bias|."""
import math

import pytest
import torch

import cdclq

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -149}
U32 = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
INF = math.inf


@pytest.fixture(scope="module")
def ctx():
    c = cdclq.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def tune():
    from cdclq import tune
    return tune


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(seed, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=rng(seed), device="cuda") * std).to(dtype)


def packed(allowed):
    """Bits of a rows x v truth table as 32-bit words."""
    m, v = allowed.shape
    words = -(-v // 32)
    bits = torch.zeros(m, words * 32, dtype=torch.int64, device="cuda")
    bits[:, :v] = allowed
    w = (bits.view(m, words, 32) << torch.arange(32, device="cuda")).sum(2)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def constraints(seed, r, v, width, nb, masks, strange=False):
    """What a batch of requests brings; with strange ids and lengths that stand for nothing."""
    g = rng(seed)
    k = {}
    if width:
        u = torch.rand(r, width, generator=g, device="cuda", dtype=torch.float64)
        k["history"] = (torch.exp(u * math.log(v + 1)) - 1).long().clamp(0, v - 1)
        k["lengths"] = torch.randint(0, width + 1, (r,), generator=g, device="cuda").int()
        k["prompts"] = (k["lengths"] * torch.rand(r, generator=g, device="cuda")).int()
        k["repetition"] = torch.rand(r, generator=g, device="cuda") + 0.5
        k["frequency"], k["presence"] = (torch.randn(r, generator=g, device="cuda") for _ in range(2))
        if strange:
            k["history"][:, ::3] = torch.tensor([-1, v, 1 << 32, -(1 << 63)], device="cuda")[
                torch.randint(0, 4, (r, len(range(0, width, 3))), generator=g, device="cuda")]
            k["lengths"][0] = width + 100
            k["prompts"][-1] = width + 7
            if r > 2:
                k["lengths"][1], k["prompts"][2] = -5, -3
    if nb:
        k["bias_tokens"] = torch.randint(0, v, (r, nb), generator=g, device="cuda")
        k["bias_tokens"][:, nb // 2:] = k["bias_tokens"][:, : nb - nb // 2]  # every token at least twice
        k["biases"] = torch.randn(r, nb, generator=g, device="cuda") * 4
        if strange:
            k["bias_tokens"][:, ::2] = -1
            k["bias_tokens"][:, 1::4] = v
    if masks:
        allowed = torch.rand(masks, v, generator=g, device="cuda") < 0.3
        allowed[0] = False  # a grammar that allows nothing
        allowed[-1, : v // 2] = True
        k["mask"] = packed(allowed)
        k["mask_rows"] = torch.randint(-1, masks, (r,), generator=g, device="cuda").int()
    return k


def wanted(logits, history=None, lengths=None, prompts=None, repetition=None, frequency=None, presence=None,
           bias_tokens=None, biases=None, mask=None, mask_rows=None):
    """The definition, request by request, in 64 bits on the host, and the magnitudes on the way."""
    out = logits.double().cpu()
    size = out.abs()
    steps = torch.zeros_like(out)
    r, v = out.shape
    for i in range(r):
        l = out[i]
        if history is not None:
            width = history.shape[1]
            n = width if lengths is None else min(max(int(lengths[i]), 0), width)
            p = 0 if prompts is None else max(int(prompts[i]), 0)
            h = history[i, :n].cpu()
            ok = (h >= 0) & (h < v)
            had = torch.unique(h[ok])
            rep = 1.0 if repetition is None else repetition[i].double().item()
            l[had] = torch.where(l[had] > 0, l[had] / rep, l[had] * rep)
            size[i, had] = torch.maximum(size[i, had], l[had].abs())
            steps[i, had] += 1
            made, c = torch.unique(h[p:][ok[p:]], return_counts=True)
            f = 0.0 if frequency is None else frequency[i].double().item()
            q = 0.0 if presence is None else presence[i].double().item()
            l[made] -= f * c + q
            size[i, made] += abs(f) * c + abs(q)
            steps[i, made] += 3
        if biases is not None:
            b = bias_tokens[i].cpu()
            ok = (b >= 0) & (b < v)
            w = biases[i].double().cpu()[ok]
            l.index_put_((b[ok],), w, accumulate=True)
            size[i].index_put_((b[ok],), w.abs(), accumulate=True)
            steps[i].index_put_((b[ok],), torch.ones(len(w), dtype=torch.float64), accumulate=True)
        if mask is not None:
            m = i if mask_rows is None else int(mask_rows[i])
            if m < -1 or m >= len(mask):
                l[:] = math.nan
            elif m >= 0:
                on = ((mask[m].cpu()[:, None] >> torch.arange(32, dtype=torch.int32)) & 1).flatten()[:v].bool()
                l[~on] = -INF
    return out, size * steps * U32


def check(got, want, bound, dtype):
    got, want = got.double().cpu(), want
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine].nan_to_num(7.0), want[~fine].nan_to_num(7.0))
    g, w = got[fine], want[fine]
    err = (g - w).abs()
    assert (err <= bound[fine] + U[dtype] * (w.abs() + bound[fine]) + TINY[dtype]).all(), err.max().item()


SIZES = [(1, 1, 1, 1, 1), (1, 31, 5, 2, 1), (3, 33, 40, 3, 2), (2, 1000, 0, 0, 2), (2, 1000, 100, 0, 0), (5, 1025, 0, 30, 0),
         (9, 5001, 300, 20, 3), (17, 8193, 2000, 300, 4), (1, 128256, 5000, 1024, 1), (70, 32000, 70, 5, 10),
         (300, 16390, 33, 4, 7), (64, 40001, 9000, 100, 9), (3, 300_000, 20_000, 70, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r,v,width,nb,masks", SIZES)
@pytest.mark.parametrize("strange", [False, True])
def test_constraints(ctx, tune, dtype, r, v, width, nb, masks, strange):
    logits = normal(r + v, r, v, std=3.0, dtype=dtype)
    k = constraints(v, r, v, width, nb, masks, strange)
    before = logits.clone()
    got = tune.constrain_logits(ctx, logits, **k)
    assert torch.equal(logits, before)
    want, bound = wanted(logits, **k)
    check(got, want, bound, dtype)
    same = (bound == 0) & torch.isfinite(want)
    assert torch.equal(got.cpu()[same], logits.cpu()[same])
    place = logits.clone()
    assert tune.constrain_logits(ctx, place, out=place, **k).data_ptr() == place.data_ptr()
    assert torch.equal(place, got)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("which", ["history", "lengths", "prompts", "repetition", "frequency", "presence", "mask_rows", "nothing"])
def test_each_by_itself(ctx, tune, dtype, which):
    """A constraint that is left out changes nothing of the others; all left out: a copy."""
    r, v = 6, 2000
    logits, k = normal(1, r, v, dtype=dtype), constraints(2, r, v, 90, 6, 6)
    keep = {"history": ["history"], "lengths": ["history", "lengths", "repetition"],
            "prompts": ["history", "prompts", "presence"], "repetition": ["history", "repetition"],
            "frequency": ["history", "frequency"], "presence": ["history", "lengths", "presence"], "mask_rows": ["mask"],
            "nothing": []}[which]
    k = {n: x for n, x in k.items() if n in keep}
    got = tune.constrain_logits(ctx, logits, **k)
    check(got, *wanted(logits, **k), dtype)
    if which in ("history", "nothing"):
        assert torch.equal(got, logits)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("place", [False, True])
def test_strides(ctx, tune, dtype, place):
    """Rows of wider tensors at odd elements; what lies beside them stays."""
    r, v, width = 5, 3001, 60
    k = constraints(3, r, v, width, 4, 3)
    k["history"] = torch.cat([k["history"], torch.zeros(r, 9, dtype=torch.int64, device="cuda")], 1)[:, :width]
    k["mask"] = torch.cat([k["mask"], k["mask"]], 1)[:, : -(-v // 32)]
    logits = normal(4, r * (v + 6) + 3, dtype=dtype)[3:].view(r, v + 6)[:, :v]
    buf = torch.zeros(r, v + 5, dtype=dtype, device="cuda")
    want = tune.constrain_logits(ctx, logits.contiguous(), **{n: x.contiguous() for n, x in k.items()})
    out = logits if place else buf[:, 2:v + 2]
    tune.constrain_logits(ctx, logits, out=out, **k)
    assert torch.equal(out, want)
    assert place or not (buf[:, :2].any() or buf[:, v + 2:].any())


@pytest.mark.parametrize("dtype", TYPES)
def test_special_values(ctx, tune, dtype):
    """Infinities, NaN and the type's lowest value: by the formula where a token is allowed, -infinity where not."""
    v = 64
    logits = torch.zeros(1, v, dtype=dtype, device="cuda")
    logits[0, :5] = torch.tensor([INF, -INF, math.nan, torch.finfo(dtype).min, torch.finfo(dtype).max])
    logits[0, 32:37] = logits[0, :5]
    allowed = torch.ones(1, v, dtype=torch.bool, device="cuda")
    allowed[0, 32:] = False
    k = dict(history=torch.arange(v, device="cuda")[None], repetition=torch.tensor([2.0], device="cuda"), mask=packed(allowed))
    got = tune.constrain_logits(ctx, logits, **k)[0]
    assert got[0] == INF and got[1] == -INF and got[2].isnan() and (got[5:32] == 0).all() and (got[32:] == -INF).all()
    assert got[3].item() == -INF and got[4].item() == torch.finfo(dtype).max / 2  # below the lowest value


@pytest.mark.parametrize("rows", [[-1, 0, 3, 1], [-2, 5, 2, 4], [1 << 30, -(1 << 31), 0, -1]])
def test_rows_of_no_mask_are_nan(ctx, tune, rows):
    v = 5000
    logits = normal(1, 4, v)
    mask = packed(torch.rand(3, v, generator=rng(2), device="cuda") < 0.5)
    at = torch.tensor(rows, dtype=torch.int32, device="cuda")
    got = tune.constrain_logits(ctx, logits, mask=mask, mask_rows=at)
    check(got, *wanted(logits, mask=mask, mask_rows=at), torch.float32)
    none = torch.full((4,), -1, dtype=torch.int32, device="cuda")
    assert torch.equal(tune.constrain_logits(ctx, logits, mask=mask[:0], mask_rows=none), logits)
    assert tune.constrain_logits(ctx, logits, mask=mask[:0], mask_rows=none + 1).isnan().all()


def test_nothing_to_do(ctx, tune):
    for r, v in ((0, 10), (0, 1)):
        assert tune.constrain_logits(ctx, normal(1, r, v)).shape == (r, v)
    logits = normal(2, 3, 100)
    empty = torch.zeros(3, 0, dtype=torch.int64, device="cuda")
    got = tune.constrain_logits(ctx, logits, history=empty, lengths=torch.zeros(3, dtype=torch.int32, device="cuda"),
                                repetition=torch.ones(3, device="cuda"), bias_tokens=empty, biases=empty.float())
    assert torch.equal(got, logits)


def test_long_histories_and_counts(ctx, tune):
    """One token 2^20 - 1 times: as many as a history holds."""
    width, v = (1 << 20) - 1, 300
    h = torch.full((1, width), 7, device="cuda")
    logits = normal(1, 1, v)
    got = tune.constrain_logits(ctx, logits, history=h, frequency=torch.tensor([2.0 ** -10], device="cuda"))
    assert got[0, 7].item() == pytest.approx(logits[0, 7].item() - width * 2.0 ** -10, rel=1e-6)
    assert torch.equal(got[0, 8:], logits[0, 8:]) and torch.equal(got[0, :7], logits[0, :7])


def test_offsets_past_32_bits(ctx, tune):
    """A history and logits whose last rows lie more than 2^32 bytes from the start."""
    r, v = 70_000, 32_001
    logits = torch.zeros(r, v, dtype=torch.bfloat16, device="cuda")
    h = torch.zeros(r, 1, dtype=torch.int64, device="cuda")
    h[-1] = v - 1
    tune.constrain_logits(ctx, logits, history=h, presence=torch.ones(r, device="cuda"), out=logits)
    assert logits[-1, -1] == -1 and logits[-1, 0] == 0 and (logits[:-1, 0] == -1).all()
    assert logits.sum(dtype=torch.float32).item() == -r


def test_captured_and_replayed(ctx, tune):
    """A decode loop: the history grows, the lengths with it."""
    r, v, width = 8, 9000, 50
    k = constraints(5, r, v, width, 5, 3)
    k["lengths"][:], k["prompts"][:] = 3, 2
    logits = normal(6, r, v, dtype=torch.bfloat16)
    tune.constrain_logits(ctx, logits, **k)
    place = logits.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = tune.constrain_logits(ctx, logits, **k)
        tune.constrain_logits(ctx, place, out=place, **k)
    for i in range(4):
        logits.copy_(normal(10 + i, r, v, dtype=torch.bfloat16))
        place.copy_(logits)
        k["lengths"].add_(10)
        k["mask_rows"].copy_(torch.randint(-1, 3, (r,), generator=rng(i), device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, place) and torch.equal(got, tune.constrain_logits(ctx, logits, **k))
        check(got, *wanted(logits, **k), torch.bfloat16)


def test_two_streams_at_once(ctx, tune):
    streams = [torch.cuda.Stream() for _ in range(2)]
    jobs = [(normal(i, 20 + i, 30_000, dtype=torch.float16), constraints(i, 20 + i, 30_000, 500, 10, 4)) for i in range(2)]
    want = [tune.constrain_logits(ctx, x, **k) for x, k in jobs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(tune.constrain_logits(ctx, jobs[i][0], **jobs[i][1]))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


def test_refusals(ctx, tune):
    r, v = 4, 100
    x, k = normal(1, r, v), constraints(2, r, v, 10, 3, 2)
    f = lambda **m: tune.constrain_logits(ctx, m.pop("logits", x), **{**k, **m})  # noqa: E731
    wide = torch.zeros(r, 1025, dtype=torch.int64, device="cuda")
    for e, m in [(TypeError, dict(logits=x.double())), (ValueError, dict(logits=x[0])), (ValueError, dict(logits=x.t())),
                 (ValueError, dict(logits=x.cpu())), (TypeError, dict(history=k["history"].int())),
                 (ValueError, dict(history=k["history"][:3])), (ValueError, dict(history=None)),
                 (TypeError, dict(lengths=k["lengths"].long())), (ValueError, dict(lengths=k["lengths"][:3])),
                 (ValueError, dict(prompts=k["prompts"][:3])), (TypeError, dict(repetition=k["repetition"].half())),
                 (ValueError, dict(frequency=k["frequency"].cpu())), (ValueError, dict(presence=k["presence"][:, None])),
                 (ValueError, dict(biases=None)), (ValueError, dict(bias_tokens=None)),
                 (ValueError, dict(biases=k["biases"][:, :2])), (TypeError, dict(biases=k["biases"].double())),
                 (ValueError, dict(bias_tokens=torch.cat([k["bias_tokens"]] * 2, 1)[:, :3])),
                 (cdclq.CdclqError, dict(bias_tokens=wide, biases=wide.float())),
                 (ValueError, dict(mask=k["mask"][:, :3])), (TypeError, dict(mask=k["mask"].long())),
                 (ValueError, dict(mask_rows=None)), (ValueError, dict(mask=None)),
                 (ValueError, dict(mask_rows=k["mask_rows"][:2])), (ValueError, dict(out=x[:3])),
                 (TypeError, dict(out=x.half())), (cdclq.CdclqError, dict(logits=x[:, :99], mask=None, mask_rows=None,
                                                                          out=x[:, 1:]))]:
        with pytest.raises(e):
            f(**m)
    with pytest.raises(cdclq.CdclqError, match="history"):
        tune.constrain_logits(ctx, x, history=torch.zeros(r, 1 << 20, dtype=torch.int64, device="cuda"))
    with pytest.raises(cdclq.CdclqError, match="vocabulary"):
        tune.constrain_logits(ctx, x[:, :0])
    h, big = torch.zeros(64, 16_000, dtype=torch.int64, device="cuda"), normal(3, 64, 20_000)
    assert cdclq.lib().cdclq_constrain_work_bytes(64, 20_000, 16_000) == 0  # looked at by every slab
    assert cdclq.lib().cdclq_constrain_work_bytes(64, 20_000, 60_000) > 4 * 64 * 60_000
    rc = cdclq.lib().cdclq_constrain_logits_device(ctx.ptr, big.data_ptr(), 20_000, 64, 20_000, cdclq.DTYPE_F32, h.data_ptr(),
                                                   16_000, 15_999 + 50_000, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, big.data_ptr(),
                                                   20_000, 0, 0, 0)
    assert rc == cdclq.INVALID_ARG  # rows of the history shorter than its width, and no workspace
    with pytest.raises(ValueError, match="without a history"):
        tune.constrain_logits(ctx, x, repetition=k["repetition"])
    assert torch.equal(x, normal(1, r, v))
