"""GPU: the training operators (attention with lse and its backward pass, rotary positions over several axes, layer and
RMS norm with modulation and their gradients) against plain implementations in 64 bits.

Tolerances are elementwise bounds of the arithmetic, made from the 64-bit reference:
  * a bf16 rounding is off by at most 2^-8 of the value (U);
  * P and dS are rounded to bf16 once before the matrix unit: each product sum is off by at most U times the sum of its
    terms' magnitudes;
  * everything else is fp32. Scores: D products of magnitudes whose scaled sum is M are off by at most D * 2^-24 * M;
    with |q| = |k| = sqrt(D) (normed heads) and scale 1 / sqrt(D), M <= sqrt(D) <= 16 and the error of a score, thus
    the relative one of P, is at most 256 * 2^-24 * 16 = 2^-12 (F).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - these tests need the MI355X box
    pytest.skip("no ROCm device", allow_module_level=True)

from f_lite import _native as nat  # noqa: E402

DEV = "cuda"
BF = torch.bfloat16
U = 2.0 ** -8
F = 2.0 ** -12
EPS = 1e-6


def close(got, ref, tol, what):
    got, ref = got.double(), ref.double()
    same = (got == ref) | (got.isnan() & ref.isnan())  # infinities
    bad = ~(((got - ref).abs() <= tol) | same)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst by "
                           f"{((got - ref).abs() / tol.clamp_min(1e-300))[bad].max().item():.3g} of the bound")


def rand(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def normed(x):
    x = x.float()
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)).to(BF)


def cu_of(lens, first=0):
    cu = [first]
    for n in lens:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, device=DEV, dtype=torch.int32)


# ------------------------------------------------------------------------------------------------ attention
def attn_ref(q, k, v, do, ql, kl, scale, q_first=0, k_first=0, f=F, u=U):
    """out, lse, dq, dk, dv in 64 bits and an elementwise bound for each, with P off by f, P and dS rounded by u; rows outside
    stay 0 (lse -inf)."""
    n, h, d = q.shape
    hk = k.shape[1]
    Q, K, V, DO = (x.double() for x in (q, k, v, do))
    ref = {x: torch.zeros_like(t) for x, t in (("out", Q), ("dq", Q), ("dk", K), ("dv", V))}
    tol = {x: torch.zeros_like(t) for x, t in ref.items()}
    ref["lse"] = torch.full((h, n), -math.inf, device=DEV, dtype=torch.float64)
    tol["lse"] = torch.full_like(ref["lse"], 2 * f)
    a, b = q_first, k_first
    for nq, nk in zip(ql, kl):
        for i in range(h if nq and nk else 0):
            j = i * hk // h
            qs, ks = slice(a, a + nq), slice(b, b + nk)
            qi, ki, vi, di = Q[qs, i], K[ks, j], V[ks, j], DO[qs, i]
            s = scale * qi @ ki.T
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.exp(s - lse)
            o = p @ vi
            ref["lse"][i, qs] = lse[:, 0]
            ref["out"][qs, i] = o
            o_err = U * o.abs() + (u + 3 * f) * (p @ vi.abs())
            tol["out"][qs, i] = o_err
            dp = di @ vi.T
            delta = (di * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            d_err = (di.abs() * o_err).sum(1, keepdim=True)  # delta is made from the rounded out
            # dS: one rounding, the error of P, and that of dP - delta
            ds_err = u * ds.abs() + 3 * f * p * (di.abs() @ vi.abs().T + delta.abs()) + p * d_err
            ref["dq"][qs, i] = scale * ds @ ki
            tol["dq"][qs, i] = abs(scale) * ds_err @ ki.abs()
            ref["dk"][ks, j] += scale * ds.T @ qi
            tol["dk"][ks, j] += abs(scale) * ds_err.T @ qi.abs()
            ref["dv"][ks, j] += p.T @ di
            tol["dv"][ks, j] += (u + 3 * f) * (p.T @ di.abs())
        a, b = a + nq, b + nk
    for x in ("dq", "dk", "dv"):
        tol[x] += U * ref[x].abs()
    for x in tol:
        tol[x] += 1e-30
    return ref, tol


ATTN = [
    # head_dim, heads, kv_heads, query lengths, key lengths
    (256, 2, 2, [1], [1]),
    (256, 2, 1, [31, 64, 1], [33, 1, 65]),
    (256, 1, 1, [129, 128, 127], [64, 63, 257]),
    (256, 3, 3, [272], [272]),
    (128, 4, 2, [5, 0, 300, 17], [200, 40, 0, 1]),
    (128, 8, 1, [140], [70]),
    (64, 6, 2, [65, 1, 1, 190], [1, 130, 600, 31]),
    (64, 1, 1, [1], [2000]),   # one query over a long context: the sweep is cut and joined
    (256, 2, 1, [9, 0, 130], [2500, 40, 33]),
    (128, 4, 1, [257, 3], [1100, 1025]),
    (64, 2, 2, [3000], [1600]),
    (64, 2, 1, [1, 3, 0, 2] * 25, [2, 0, 5, 40] * 25),  # more sequences than a wave has lanes
    (64, 1, 1, [1, 3, 0, 130, 2] * 210, [2, 0, 5, 140, 1] * 210),  # work lists of more than 64 x 64 entries
    (64, 4, 4, [1500], [3]),
    (256, 12, 12, [700], [77]),
]


def attn_inputs(d, h, hk, ql, kl, seed=0, first=0, behind=0):
    lq, lk = sum(ql) + first + behind, sum(kl) + first + behind
    common = rand(1, 1, d, seed=seed + 9)
    q = normed(rand(lq, h, d, seed=seed) + 0.5 * common)
    k = normed(rand(lk, hk, d, seed=seed + 1) + 0.5 * common)
    return q, k, rand(lk, hk, d, seed=seed + 2, dtype=BF), rand(lq, h, d, seed=seed + 3, dtype=BF)


@pytest.mark.parametrize("d,h,hk,ql,kl", ATTN)
def test_attention_forward_backward(d, h, hk, ql, kl):
    q, k, v, do = attn_inputs(d, h, hk, ql, kl)
    cq, ck, scale = cu_of(ql), cu_of(kl), d ** -0.5
    ref, tol = attn_ref(q, k, v, do, ql, kl, scale)
    out, lse = nat.attn_varlen_lse(q, k, v, cq, ck, scale)
    close(out, ref["out"], tol["out"], "out")
    close(lse, ref["lse"], tol["lse"], "lse")
    grads = nat.attn_varlen_bwd(do, q, k, v, out, lse, cq, ck, scale)
    for x, g in zip(("dq", "dk", "dv"), grads):
        close(g, ref[x], tol[x], x)
    again = nat.attn_varlen_bwd(do, q, k, v, out, lse, cq, ck, scale)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_strided_and_rows_outside(d):
    """q, k, v as slices of one qkv tensor (gradients into slices of another), head-major out, and packed batches that
    begin after row 0 and end before the last row: those rows stay, or are zeros in tensors made by the call. They hold
    NaN, which nothing may read."""
    h, ql, kl, first, behind = 2, [70, 0, 33], [70, 5, 33], 3, 40
    q, k, v, do = attn_inputs(d, h, h, ql, kl, seed=4, first=first, behind=behind)
    n_q, n_k = q.shape[0], k.shape[0]
    rows = max(n_q, n_k)
    qkv = torch.full((rows, 3 * h + 1, d), math.nan, device=DEV, dtype=BF)
    for t, at in ((q, 0), (k, h), (v, 2 * h)):
        n = t.shape[0]
        qkv[first:n - behind, at:at + h] = t[first:n - behind]
    Q, K, V = qkv[:n_q, :h], qkv[:n_k, h:2 * h], qkv[:n_k, 2 * h:3 * h]
    do = do.transpose(0, 1).contiguous().transpose(0, 1)  # head-major
    do[:first], do[n_q - behind:] = math.nan, math.nan
    cq, ck, scale = cu_of(ql, first), cu_of(kl, first), d ** -0.5
    ref, tol = attn_ref(q, k, v, do.nan_to_num(), ql, kl, scale, first, first)
    out, lse = nat.attn_varlen_lse(Q, K, V, cq, ck, scale)
    out_hm = torch.full((h, n_q, d), 7.0, device=DEV, dtype=BF).transpose(0, 1)
    lse2 = torch.full((h, n_q), 7.0, device=DEV)
    nat.attn_varlen_lse(Q, K, V, cq, ck, scale, out=out_hm, lse=lse2)
    outside = torch.ones(n_q, dtype=torch.bool, device=DEV)
    outside[first:n_q - behind] = False
    assert (out[outside] == 0).all() and (lse[:, outside] == -math.inf).all()
    assert (out_hm[outside] == 7).all() and (lse2[:, outside] == 7).all()
    assert torch.equal(out[~outside], out_hm[~outside]) and torch.equal(lse[:, ~outside], lse2[:, ~outside])
    close(out, ref["out"], tol["out"], "out")
    grads = nat.attn_varlen_bwd(do, Q, K, V, out_hm, lse, cq, ck, scale)
    for x, g in zip(("dq", "dk", "dv"), grads):
        close(g, ref[x], tol[x], x)
    buf = torch.full_like(qkv, 5.0)
    into = buf[:n_q, :h], buf[:n_k, h:2 * h], buf[:n_k, 2 * h:3 * h]
    nat.attn_varlen_bwd(do, Q, K, V, out_hm, lse, cq, ck, scale, *into)
    for g, t in zip(grads, into):
        n = t.shape[0]
        assert torch.equal(t[first:n - behind], g[first:n - behind])
        assert (t[:first] == 5).all() and (t[n - behind:] == 5).all()
        assert (g[:first] == 0).all() and (g[n - behind:] == 0).all()
    assert (buf[:, 3 * h:] == 5).all()


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_attention_far_scores(d, sign):
    """All scores near -1000 (or 1000), lengths that end inside a tile: exp(-lse) of a padding key would overflow."""
    ql, kl = [70], [37]
    q, k, v, do = attn_inputs(d, 1, 1, ql, kl, seed=8)
    q[..., 0], k[..., 0] = 32.0, sign * 32.0
    cq, ck, scale = cu_of(ql), cu_of(kl), 1.0
    # scores of up to ~1300 in fp32: D * 2^-24 * 1300 * 2 relative error of P
    ref, tol = attn_ref(q, k, v, do, ql, kl, scale)
    slack = d * 2.0 ** -24 * 1300 * 2 / F
    p_err = {x: slack * F for x in tol}
    out, lse = nat.attn_varlen_lse(q, k, v, cq, ck, scale)
    grads = nat.attn_varlen_bwd(do, q, k, v, out, lse, cq, ck, scale)
    # the same bounds with the larger error of P: at most slack times all of each bound's P terms
    for x, g in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        assert torch.isfinite(g).all(), x
        close(g, ref[x], tol[x] * (1 + p_err[x] / U) + slack * F * (abs(ref[x]) if x == "lse" else 1e-9), x)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("scale", [1.0, -1.0, 0.0])
@pytest.mark.parametrize("ql,kl", [([70, 300], [500, 129]), ([3, 5], [500, 129]), ([2, 130], [4000, 600])])
def test_attention_scores_that_grow(d, scale, ql, kl):
    """The largest score of some queries comes late and is far above the first ones (up to e^300); a negative scale turns
    the order round, with a scale of zero all keys count alike. With 2 queries and 4000 keys the sweep is cut."""
    q, k, v, do = attn_inputs(d, 2, 1, ql, kl, seed=12)
    q, k = (q.float() * 0.05).to(BF), (k.float() * 0.05).to(BF)
    q[..., 0] = 4.0
    k[..., 0] = 0.0
    k[400:, :, 0], k[490:, :, 0], k[600:, :, 0] = 40.0, 75.0, -30.0
    cq, ck = cu_of(ql), cu_of(kl)
    # scores of up to 300, one product of 300 and small ones that sum to under 2: off by at most d * 2^-24 * 302
    ref, tol = attn_ref(q, k, v, do, ql, kl, scale, f=F + d * 2.0 ** -24 * 302)
    out, lse = nat.attn_varlen_lse(q, k, v, cq, ck, scale)
    grads = nat.attn_varlen_bwd(do, q, k, v, out, lse, cq, ck, scale)
    for x, g in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        close(g, ref[x], tol[x], x)


@pytest.mark.parametrize("d,h,hk,ql,kl", [
    (64, 1, 1, [1], [3]), (128, 1, 1, [2], [5]), (256, 1, 1, [1], [2]),
    (64, 4, 2, [1, 3, 0, 7, 16], [2, 90, 5, 33, 31]),
    (128, 2, 1, [32, 1, 31], [32, 33, 3]),
    (256, 4, 2, [1, 3, 0, 7, 16], [2, 90, 5, 33, 31]),
    (64, 2, 1, [128], [512]), (64, 2, 1, [2000], [5]), (128, 1, 1, [64], [40]), (256, 2, 2, [1], [4000]),
])
def test_attention_of_few_rows(d, h, hk, ql, kl):
    """Few probabilities or results: P and dS count with what bf16 drops of them (fp16, or two bf16 parts)."""
    cq, ck, scale = cu_of(ql), cu_of(kl), d ** -0.5
    for seed in range(4):
        q, k, v, do = attn_inputs(d, h, hk, ql, kl, seed=30 + 10 * seed)
        ref, tol = attn_ref(q, k, v, do, ql, kl, scale, u=2.0 ** -12)
        out, lse = nat.attn_varlen_lse(q, k, v, cq, ck, scale)
        grads = nat.attn_varlen_bwd(do, q, k, v, out, lse, cq, ck, scale)
        pairs = max(a * b for a, b in zip(ql, kl)) * h
        for x, g in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
            few = pairs <= 2048 or max(ql) * h * d <= 8192 if x == "out" else pairs <= 2 ** 17 or max(kl) * hk * d <= 32768
            if few or x in ("lse", "dq"):
                close(g, ref[x], tol[x], x)


def test_attention_gradients_against_differences():
    d, ql, kl = 64, [40, 9], [21, 50]
    q, k, v, do = attn_inputs(d, 2, 1, ql, kl, seed=3)
    cq, ck, scale = cu_of(ql), cu_of(kl), d ** -0.5
    out, lse = nat.attn_varlen_lse(q, k, v, cq, ck, scale)
    grads = nat.attn_varlen_bwd(do, q, k, v, out, lse, cq, ck, scale)

    def loss(q, k, v):
        total, a, b = 0.0, 0, 0
        for n, m in zip(ql, kl):
            for i in range(2):
                p = torch.softmax(scale * q[a:a + n, i] @ k[b:b + m, 0].T, 1)
                total = total + ((p @ v[b:b + m, 0]) * do[a:a + n, i].double()).sum()
            a, b = a + n, b + m
        return total

    base = [x.double() for x in (q, k, v)]
    _, tol = attn_ref(q, k, v, do, ql, kl, scale)
    for which, (g, x) in enumerate(zip(grads, ("dq", "dk", "dv"))):
        u = rand(*g.shape, seed=20 + which).double()
        step = 1e-4
        ends = []
        for sg in (step, -step):
            at = list(base)
            at[which] = at[which] + sg * u
            ends.append(loss(*at))
        diff = (ends[0] - ends[1]) / (2 * step)
        bound = (tol[x] * u.abs()).sum() + 1e-5 * (g.double() * u).abs().sum()
        assert abs((g.double() * u).sum() - diff) <= bound, x


def test_attention_refusals():
    q, k, v, do = attn_inputs(64, 4, 2, [8], [8])
    cu = cu_of([8])
    out, lse = nat.attn_varlen_lse(q, k, v, cu, cu, 0.1)
    bad = [
        lambda: nat.attn_varlen_lse(q.float(), k, v, cu, cu, 0.1),
        lambda: nat.attn_varlen_lse(q, k[:, :, :32], v[:, :, :32], cu, cu, 0.1),
        lambda: nat.attn_varlen_lse(q[:, :3], k, v, cu, cu, 0.1),
        lambda: nat.attn_varlen_lse(q, k, v[:4], cu, cu, 0.1),
        lambda: nat.attn_varlen_lse(q, k[:1].expand(8, 2, 64), v, cu, cu, 0.1),  # expanded rows
        lambda: nat.attn_varlen_lse(q, k, v, cu.long(), cu, 0.1),
        lambda: nat.attn_varlen_lse(q, k, v, cu, cu_of([4, 4]), 0.1),
        lambda: nat.attn_varlen_lse(q, k, v, cu[:1], cu[:1], 0.1),
        lambda: nat.attn_varlen_lse(q, k, v, cu.cpu(), cu, 0.1),
        lambda: nat.attn_varlen_lse(q, k, v, cu, cu, 0.1, out=torch.empty_like(q)),  # out without lse
        lambda: nat.attn_varlen_lse(q, k, v, cu, cu, 0.1, out=out[:, :1].expand(8, 4, 64), lse=lse),
        lambda: nat.attn_varlen_bwd(do, q, k, v, out, lse.T.contiguous(), cu, cu, 0.1),
        lambda: nat.attn_varlen_bwd(do.sum().to(BF).expand(8, 4, 64), q, k, v, out, lse, cu, cu, 0.1),
        lambda: nat.attn_varlen_bwd(do, q, k, v, out, lse, cu, cu, 0.1, dq=torch.empty_like(q)),
        lambda: nat.attn_varlen_bwd(do.float(), q, k, v, out, lse, cu, cu, 0.1),
    ]
    for call in bad:
        with pytest.raises(nat.FliteError):
            call()
    # heads that share their data are fine as inputs
    ke, ve = k[:, :1].expand(8, 2, 64), v[:, :1].expand(8, 2, 64)
    o2, _ = nat.attn_varlen_lse(q, ke, ve, cu, cu, 0.1)
    o3, _ = nat.attn_varlen_lse(q, ke.contiguous(), ve.contiguous(), cu, cu, 0.1)
    assert torch.equal(o2, o3)


def test_attention_empty():
    for ql, kl in (([0], [5]), ([5], [0]), ([0], [0])):
        q, k, v, do = attn_inputs(64, 2, 2, ql, kl)
        cq, ck = cu_of(ql), cu_of(kl)
        out, lse = nat.attn_varlen_lse(q, k, v, cq, ck, 0.1)
        grads = nat.attn_varlen_bwd(do, q, k, v, out, lse, cq, ck, 0.1)
        assert (out == 0).all() and (lse == -math.inf).all() and all((g == 0).all() for g in grads)


# ------------------------------------------------------------------------------------------------ rotary positions
def rope_ref(x, pos, pairs, base, interleaved, norm, rope_heads, back=None):
    """Forward (out, rstd, bound), or with back = (y, rstd) the gradient of x from the gradient x, in 64 bits."""
    x = x.double()
    rows, h, d = x.shape
    n = sum(pairs)
    freq = torch.cat([float(b) ** (-torch.arange(m, dtype=torch.float64) / max(m, 1)) for m, b in zip(pairs, base)]).to(DEV)
    ax = torch.tensor([a for a, m in enumerate(pairs) for _ in range(m)], device=DEV)
    ang = pos.double()[:, ax] * freq
    ang = ang.repeat(rows // max(pos.shape[0], 1), 1)[:, None]
    c, s = ang.cos(), ang.sin()
    mag = x.abs()
    if back is not None:
        s = -s
        if norm:
            y, r = back[0].double(), back[1].double()[..., None]
            dot = (x * y).mean(-1, keepdim=True)
            mag = r * (x.abs() + y.abs() * (x * y).abs().mean(-1, keepdim=True))
            x = r * (x - y * dot)

    def turn(t, c, s):
        out = t.clone()
        i1 = torch.arange(n, device=DEV) * 2 if interleaved else torch.arange(n, device=DEV)
        i2 = i1 + 1 if interleaved else i1 + n
        t1, t2 = t[:, :rope_heads, i1], t[:, :rope_heads, i2]
        out[:, :rope_heads, i1], out[:, :rope_heads, i2] = t1 * c + t2 * s, t2 * c - t1 * s
        return out

    y = turn(x, c, s)
    # fp32: the sines are off by 2^-22, each product and sum by 2^-24 of its magnitude, the mean by < 16 of them
    mag = turn(mag, torch.ones_like(c), torch.ones_like(s))
    mag[:, :rope_heads] = mag[:, :rope_heads].abs() + 2 * mag[:, :rope_heads].abs().amax(-1, keepdim=True)
    err = 2.0 ** -20 * mag
    if back is not None or not norm:
        return y, None, err
    r = torch.rsqrt(y.square().mean(-1) + EPS)
    return y * r[..., None], r, err * r[..., None]


ROPE = [
    # tokens (frames, height, width), repeats, heads, head_dim, pairs, bases, interleaved, rope_heads
    ((1, 1, 1), 1, 1, 64, (32,), 1e4, False, None),
    ((3, 5, 7), 2, 3, 128, (16, 24, 24), 1e4, True, None),
    ((3, 5, 7), 1, 5, 128, (22, 21, 21), (100.0, 1e4, 5e5), False, 2),
    ((1, 6, 6), 2, 24, 256, (64, 64), 1e4, False, None),
    ((2, 3, 3), 1, 2, 256, (1, 3, 4), 1e4, True, None),     # most of the head is not turned
    ((1, 9, 4), 1, 8, 64, (0, 8, 8), 1e4, False, 0),          # nothing is turned
    ((4, 4, 4), 1, 40, 48, (2, 6, 8), 1e4, True, 39),         # 48 is no power of two
    ((1, 33, 9), 1, 1, 16, (0, 4, 4), 1e4, False, None),
]


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("grid,rep,h,d,pairs,base,inter,rope_heads", ROPE)
def test_rope_axes(grid, rep, h, d, pairs, base, inter, rope_heads, dtype, norm):
    t = torch.stack(torch.meshgrid(*[torch.arange(n) for n in grid], indexing="ij"), -1).reshape(-1, 3)
    t = t[:, 3 - len(pairs):] + torch.tensor([100000, 0, -3][3 - len(pairs):])
    pos = t.to(DEV, torch.int32)
    tokens, rows = pos.shape[0], pos.shape[0] * rep
    wide = rand(rows, h + 2, d, seed=rows, dtype=dtype)
    x = wide[:, 1:1 + h]  # a slice of wider rows
    keep = wide.clone()
    bases = base if isinstance(base, tuple) else (base,) * len(pairs)
    rh = h if rope_heads is None else rope_heads
    ulp = U if dtype == BF else 2.0 ** -24
    ref, r_ref, err = rope_ref(x, pos, pairs, bases, inter, norm, rh)
    y, r = nat.rope_axes(x, pos, pairs, base, interleaved=inter, norm=norm, rope_heads=rope_heads)
    close(y, ref, ulp * ref.abs() + err + 1e-30, "y")
    if norm:
        close(r, r_ref, 2.0 ** -20 * r_ref, "rstd")
    else:
        assert r is None
    fp = nat.rope_axes(x, pos.float(), pairs, base, interleaved=inter, norm=norm, rope_heads=rope_heads)[0]
    assert torch.equal(fp, y)  # the positions are whole: exact in fp32
    dy = rand(rows, h, d, seed=5, dtype=dtype)
    back = (y, r) if norm else None
    ref, _, err = rope_ref(dy, pos, pairs, bases, inter, norm, rh, back=back or ())
    dx = nat.rope_axes_bwd(dy, pos, pairs, base, interleaved=inter, y=y if norm else None, rstd=r,
                           rope_heads=rope_heads)
    close(dx, ref, ulp * ref.abs() + err + 1e-30, "dx")
    # in place, forward and backward
    y2, r2 = nat.rope_axes(x, pos, pairs, base, interleaved=inter, norm=norm, rope_heads=rope_heads, out=x)
    assert y2 is x and torch.equal(x, y) and (not norm or torch.equal(r, r2))
    assert torch.equal(wide[:, 0], keep[:, 0]) and torch.equal(wide[:, 1 + h:], keep[:, 1 + h:])
    dy2 = dy.clone()
    nat.rope_axes_bwd(dy2, pos, pairs, base, interleaved=inter, y=y if norm else None, rstd=r, rope_heads=rope_heads,
                      out=dy2)
    assert torch.equal(dy2, dx)


def test_rope_axes_is_the_models_rope():
    """Two axes of 64 pairs, registers at position 0: rope_qknorm_ with the model's tables."""
    hh, ww, reg, h = 5, 7, 16, 3
    cos, sin = nat.rope_tables(hh, ww, reg, round_bf16=False)
    grid = torch.stack(torch.meshgrid(torch.arange(hh), torch.arange(ww), indexing="ij"), -1).reshape(-1, 2)
    pos = torch.cat([torch.zeros(reg, 2, dtype=torch.long), grid]).to(DEV, torch.int32)
    x = rand(2 * (reg + hh * ww), h, 256, dtype=BF)
    ref = nat.rope_qknorm_(x.clone().view(x.shape[0], -1), h, h, cos, sin, reg + hh * ww).view_as(x)
    y, _ = nat.rope_axes(x, pos, (64, 64), norm=True)
    # Both sides are rounded once: with a and b the values before, |y - ref| <= U |a| + U |b| + |a - b|, so two
    # half steps (neighbouring bf16 values differ by a whole one, 2 U). |a - b|: the tables' fp32 angles are off by up
    # to 7 * 2^-24 at |y| <= 16, and U of it
    close(y, ref, 2 * U * ref.double().abs() + 2.0 ** -16, "y")


def test_rope_axes_gradient_against_differences():
    pos = torch.tensor([[0, 0], [1, 3], [70000, -2]], device=DEV, dtype=torch.int32)
    x, dy = rand(3, 2, 32, seed=1), rand(3, 2, 32, seed=2)
    y, r = nat.rope_axes(x, pos, (5, 11), norm=True)
    dx = nat.rope_axes_bwd(dy, pos, (5, 11), y=y, rstd=r).double()
    u = rand(3, 2, 32, seed=3).double()
    f = lambda t: (rope_ref(t, pos, (5, 11), (1e4, 1e4), False, True, 2)[0] * dy.double()).sum()  # noqa: E731
    diff = (f(x.double() + 1e-5 * u) - f(x.double() - 1e-5 * u)) / 2e-5
    # dx is off by 2^-18 of magnitudes of at most |dy| + |y| mean|y dy| <= 10 (fp32); differences by 1e-8
    assert abs((dx * u).sum() - diff) <= 2.0 ** -18 * 10 * u.abs().sum()


def test_rope_axes_refusals():
    x, pos = rand(6, 2, 64, dtype=BF), torch.zeros(3, 2, device=DEV, dtype=torch.int32)
    y, r = nat.rope_axes(x, pos, (16, 16), norm=True)
    for call in (
            lambda: nat.rope_axes(x.half(), pos, (16, 16)), lambda: nat.rope_axes(x[0], pos, (16, 16)),
            lambda: nat.rope_axes(x, pos.long(), (16, 16)), lambda: nat.rope_axes(x, pos, (16, 16, 0)),
            lambda: nat.rope_axes(x, pos, (16, 17)), lambda: nat.rope_axes(x, pos, (16, 24)),
            lambda: nat.rope_axes(x[:5], pos, (16, 16)), lambda: nat.rope_axes(x, pos[:0], (16, 16)),
            lambda: nat.rope_axes(x, pos, (16, 16), base=(1e4,)), lambda: nat.rope_axes(x, pos, (16, 16), base=-1.0),
            lambda: nat.rope_axes(x, pos, (16, 16), rope_heads=3),
            lambda: nat.rope_axes(x, pos, (16, 16), out=x.float()),
            lambda: nat.rope_axes(x, pos, (16, 16), out=x[:, :1].expand(6, 2, 64)),
            lambda: nat.rope_axes(x, pos.cpu(), (16, 16)),
            lambda: nat.rope_axes_bwd(x, pos, (16, 16), y=y), lambda: nat.rope_axes_bwd(x, pos, (16, 16), rstd=r),
            lambda: nat.rope_axes_bwd(x, pos, (16, 16), y=y[:3], rstd=r),
            lambda: nat.rope_axes_bwd(x, pos, (16, 16), y=y, rstd=r.T.contiguous())):
        with pytest.raises(nat.FliteError):
            call()
    assert nat.rope_axes(x[:0], pos, (16, 16), norm=True)[0].shape == (0, 2, 64)


# ------------------------------------------------------------------------------------------------ norms
def norm_ref(x, w, b, shift, scale, seg_rows, rms, dy=None):
    """64-bit forward pass (y, bound), or with dy all gradients and their bounds."""
    X = x.double()
    rows, d = X.shape
    seg = torch.arange(rows, device=DEV) // (seg_rows or max(rows, 1))
    segs = (rows + seg_rows - 1) // seg_rows if seg_rows else 1
    mean = X.mean(1, keepdim=True) * (0 if rms else 1)
    r = torch.rsqrt((X - mean).square().mean(1, keepdim=True) + EPS)
    n = (X - mean) * r
    # fp32: the mean is a sum of d terms in a tree of less than 2^5 steps: off by 2^-19 of the row's largest |x|, so n by
    # that times r; the same for the deviation
    n_err = 2.0 ** -18 * (X.abs().amax(1, keepdim=True) * r + n.abs())
    one = torch.ones(d, device=DEV, dtype=torch.float64)
    W, B = one if w is None else w.double(), 0 * one if b is None else b.double()
    rows_of = lambda m: 0 if m is None else (m.double()[seg] if m.dim() == 2 else m.double())  # noqa: E731
    g1 = 1 + rows_of(scale)
    if dy is None:
        y = (n * W + B) * g1 + rows_of(shift)
        return y, U * y.abs() + n_err * (W * g1).abs() + 2.0 ** -20 * (B * g1).abs()
    DY = dy.double()
    g = DY * W * g1
    c1, c2 = g.mean(1, keepdim=True) * (0 if rms else 1), (g * n).mean(1, keepdim=True)
    dx = r * (g - c1 - n * c2)
    c2_err = (g.abs() * n_err).mean(1, keepdim=True) + 2.0 ** -19 * (g * n).abs().mean(1, keepdim=True)
    dx_err = r * (2.0 ** -19 * (g.abs() + g.abs().mean(1, keepdim=True) + (n * c2).abs()) + n_err * c2.abs()
                  + n.abs() * c2_err) + 2.0 ** -18 * dx.abs()
    zeros = torch.zeros(segs, d, device=DEV, dtype=torch.float64)
    # sums over rows: at most 2^7 sequential steps per level, 2^-17 of the sum of magnitudes, and the error of n
    at = lambda t: zeros.index_add(0, seg, t)  # noqa: E731
    nb, nb_err = n * W + B, n_err * W.abs()
    ref = {"dx": dx, "dshift": at(DY), "dscale": at(DY * nb), "dw": (DY * g1 * n).sum(0), "db": (DY * g1).sum(0)}
    s = 2.0 ** -16
    tol = {"dx": dx_err, "dshift": s * at(DY.abs()), "dscale": at(DY.abs() * (s * ((n * W).abs() + B.abs()) + nb_err)),
           "dw": (DY * g1).abs().mul(s * n.abs() + n_err).sum(0), "db": s * (DY * g1).abs().sum(0)}
    return ref, tol


NORM = [
    # rows, dim, seg_rows, affine, modulation ("none", "rows": one per segment, "one": a single row)
    (1, 8, 0, True, "one"),
    (5, 64, 2, True, "rows"),
    (77, 520, 30, False, "rows"),
    (130, 1024, 0, True, "none"),
    (33, 4096, 16, True, "rows"),
    (9, 4104, 4, True, "rows"),
    (6, 8192, 0, False, "none"),
    (300, 256, 1, True, "rows"),      # every row its own segment
    (700, 72, 100, True, "one"),
    (2100, 640, 1000, True, "rows"),
]


def norm_inputs(rows, d, seg_rows, affine, mod, dtype, rms, seed=0):
    segs = (rows + seg_rows - 1) // seg_rows if seg_rows else 1
    wide = rand(rows, d + 8, seed=seed).mul_(1.5).add_(2.0).to(dtype)  # a mean that is not small
    x = wide[:, :d]
    w = (1 + 0.2 * rand(d, seed=seed + 1)).to(BF) if affine else None
    b = (0.3 * rand(d, seed=seed + 2)).to(BF) if affine and not rms else None
    shape = {"none": None, "rows": (segs, d), "one": (d,)}[mod]
    mods = [None if shape is None else 0.3 * rand(*shape, seed=seed + 3 + i) for i in range(2)]
    return x, w, b, mods[0], mods[1], rand(rows, d, seed=seed + 6, dtype=BF)


@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("rows,d,seg_rows,affine,mod", NORM)
def test_layernorm_modulate(rows, d, seg_rows, affine, mod, dtype):
    x, w, b, shift, scale, _ = norm_inputs(rows, d, seg_rows, affine, mod, dtype, False)
    y = nat.layernorm_modulate(x, w, b, shift, scale, seg_rows)
    ref, tol = norm_ref(x, w, b, shift, scale, seg_rows, False)
    close(y, ref, tol, "y")
    buf = torch.full((rows, d + 16), 3.0, device=DEV, dtype=BF)
    nat.layernorm_modulate(x, w, b, shift, scale, seg_rows, out=buf[:, 8:8 + d])
    assert torch.equal(buf[:, 8:8 + d], y) and (buf[:, :8] == 3).all() and (buf[:, 8 + d:] == 3).all()


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("rows,d,seg_rows,affine,mod", NORM)
def test_norm_modulate_bwd(rows, d, seg_rows, affine, mod, dtype, rms):
    x, w, b, shift, scale, dy = norm_inputs(rows, d, seg_rows, affine, mod, dtype, rms)
    ref, tol = norm_ref(x, w, b, shift, scale, 0 if mod == "one" else seg_rows, rms, dy)
    got = dict(zip(("dx", "dw", "db", "dshift", "dscale"),
                   nat.norm_modulate_bwd(dy, x, w, b, scale, seg_rows, rms=rms)))
    assert got["dx"].dtype == dtype
    tol["dx"] = tol["dx"] + (U if dtype == BF else 2.0 ** -24) * ref["dx"].abs()
    present = {"dx": True, "dw": w is not None, "db": b is not None, "dshift": scale is not None,
               "dscale": scale is not None}
    for name, want in present.items():
        assert (got[name] is not None) == want, name
        if want:
            assert name == "dx" or got[name].dtype == torch.float32
            if mod == "one" and name in ("dshift", "dscale"):
                assert got[name].shape == (d,)
            close(got[name].view_as(ref[name]), ref[name], tol[name] + 1e-30, name)
    again = nat.norm_modulate_bwd(dy, x, w, b, scale, seg_rows, rms=rms)
    assert all(a is None or torch.equal(a, g) for a, g in zip(again, got.values()))
    dx = torch.full((rows, d + 16), 3.0, device=DEV, dtype=dtype)
    nat.norm_modulate_bwd(dy, x, w, b, scale, seg_rows, rms=rms, dx=dx[:, 8:8 + d])
    assert torch.equal(dx[:, 8:8 + d], got["dx"]) and (dx[:, :8] == 3).all() and (dx[:, 8 + d:] == 3).all()


def test_norm_shift_alone_and_rms_forward_agree():
    x, w, _, shift, _, dy = norm_inputs(50, 256, 20, True, "rows", torch.float32, True)
    got = nat.norm_modulate_bwd(dy, x, w, seg_rows=20, rms=True, shift=True)
    ref, tol = norm_ref(x, w, None, shift, None, 20, True, dy)
    assert got[4] is None
    close(got[3], ref["dshift"], tol["dshift"], "dshift")
    y = nat.rmsnorm_modulate(x, w, shift, None, seg_rows=20)
    ref, tol = norm_ref(x, w, None, shift, None, 20, True)
    close(y, ref, tol, "y")


@pytest.mark.parametrize("rms", [False, True])
def test_norm_gradient_against_differences(rms):
    x, w, b, shift, scale, dy = norm_inputs(7, 64, 3, True, "rows", torch.float32, rms)
    got = nat.norm_modulate_bwd(dy, x, w, b, scale, 3, rms=rms)
    ref_tol = norm_ref(x, w, b, shift, scale, 3, rms, dy)[1]
    seg = torch.arange(7, device=DEV) // 3

    def loss(x, w, b, shift, scale):
        m = 0 if rms else x.mean(1, keepdim=True)
        n = (x - m) * torch.rsqrt((x - m).square().mean(1, keepdim=True) + EPS)
        return (((n * w + b) * (1 + scale[seg]) + shift[seg]) * dy.double()).sum()

    ins = [x, w, torch.zeros(64, device=DEV) if b is None else b, shift, scale]
    ins = [t.double() for t in ins]
    for i, (g, name) in enumerate(zip(got, ("dx", "dw", "db", "dshift", "dscale"))):
        if g is None:
            continue
        u = rand(*g.shape, seed=40 + i).double()
        ends = [loss(*[t + sg * u if j == i else t for j, t in enumerate(ins)]) for sg in (1e-5, -1e-5)]
        bound = (ref_tol[name] * u.abs()).sum() + 1e-7 * (g.double() * u).abs().sum()
        assert abs((g.double() * u).sum() - (ends[0] - ends[1]) / 2e-5) <= bound, name


def test_norm_refusals_and_empty():
    x, w, b, shift, scale, dy = norm_inputs(8, 64, 4, True, "rows", BF, False)
    f, g = nat.layernorm_modulate, nat.norm_modulate_bwd
    for call in (lambda: f(x.half(), w), lambda: f(x[:, :60]), lambda: f(x, w.float()), lambda: f(x, w[:32]),
                 lambda: f(x, w, b, shift[:1], scale, 4), lambda: f(x, w, b, shift.double(), scale, 4),
                 lambda: f(x, w, b, shift, scale, -1), lambda: f(x[:1].expand(8, 64)), lambda: f(x.t()),
                 lambda: f(x, w, b, shift, scale, 4, out=torch.empty(8, 64, device=DEV)),
                 lambda: g(dy.float(), x), lambda: g(dy[:4], x), lambda: g(dy, x, w, b, rms=True),
                 lambda: g(dy, x, w, b, scale, 3), lambda: g(dy, x, dx=torch.empty(8, 64, device=DEV)),
                 lambda: g(dy, x, w.cpu())):
        with pytest.raises(nat.FliteError):
            call()
    assert f(x[:0], w, b).shape == (0, 64)
    dx, dw, db, _, _ = g(dy[:0], x[:0], w, b)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()


# ------------------------------------------------------------------------------------------------ together
def block(x, w, b, shift, scale, wqkv, pos, pairs, cu, h, d):
    """Norm -> qkv -> rotary positions + per-head norm -> attention, keeping what the way back needs."""
    rows = x.shape[0]
    seg = pos.shape[0]
    n = nat.layernorm_modulate(x, w, b, shift, scale, seg)
    qkv = nat.gemm(n, wqkv).view(rows, 3 * h, d)
    qk, rstd = nat.rope_axes(qkv[:, :2 * h], pos, pairs, norm=True, out=qkv[:, :2 * h])
    out, lse = nat.attn_varlen_lse(qkv[:, :h], qkv[:, h:2 * h], qkv[:, 2 * h:], cu, cu, d ** -0.5)
    return n, qkv, rstd, out, lse


def block_bwd(do, x, w, b, scale, wqkv, pos, pairs, cu, h, d, n, qkv, rstd, out, lse):
    rows = x.shape[0]
    dqkv = torch.empty_like(qkv)
    nat.attn_varlen_bwd(do, qkv[:, :h], qkv[:, h:2 * h], qkv[:, 2 * h:], out, lse, cu, cu, d ** -0.5,
                        dqkv[:, :h], dqkv[:, h:2 * h], dqkv[:, 2 * h:])
    nat.rope_axes_bwd(dqkv[:, :2 * h], pos, pairs, y=qkv[:, :2 * h], rstd=rstd, out=dqkv[:, :2 * h])
    dn = nat.gemm(dqkv.view(rows, -1), wqkv.t().contiguous())
    return (dqkv,) + nat.norm_modulate_bwd(dn, x, w, b, scale, pos.shape[0])


def block_setup(seed=0):
    h, d, dim, pairs = 2, 256, 512, (64, 64)
    reg, hh, ww, batch = 16, 6, 9, 2
    grid = torch.stack(torch.meshgrid(torch.arange(hh), torch.arange(ww), indexing="ij"), -1).reshape(-1, 2)
    pos = torch.cat([torch.zeros(reg, 2, dtype=torch.long), grid]).to(DEV, torch.int32)
    seg = pos.shape[0]
    rows = batch * seg
    x = rand(rows, dim, seed=seed, dtype=BF)
    w, b = (1 + 0.1 * rand(dim, seed=seed + 1)).to(BF), (0.1 * rand(dim, seed=seed + 2)).to(BF)
    shift, scale = 0.2 * rand(batch, dim, seed=seed + 3), 0.2 * rand(batch, dim, seed=seed + 4)
    wqkv = (rand(3 * h * d, dim, seed=seed + 5) * dim ** -0.5).to(BF)
    do = rand(rows, h, d, seed=seed + 6, dtype=BF)
    return x, w, b, shift, scale, wqkv, pos, pairs, cu_of([seg] * batch), h, d, do


def test_attention_branch_forward_and_backward():
    """The attention branch of a block against autograd in 64 bits. Each stored tensor is rounded to bf16 once: n, qkv,
    the turned heads, P, out, dS, the gradients of q, k, v, of the turn, dn and dx: 12 roundings of at most 2^-8 each in
    the relative norm (the steps between them are linear maps or norms, whose condition here is below 2)."""
    x, w, b, shift, scale, wqkv, pos, pairs, cu, h, d, do = block_setup()
    saved = block(x, w, b, shift, scale, wqkv, pos, pairs, cu, h, d)
    grads = block_bwd(do, x, w, b, scale, wqkv, pos, pairs, cu, h, d, *saved)
    leaves = [t.double().requires_grad_() for t in (x, w, b, shift, scale)]
    X, W, B, SH, SC = leaves
    rows, seg = x.shape[0], pos.shape[0]
    mean = X.mean(1, keepdim=True)
    n = (X - mean) * torch.rsqrt((X - mean).square().mean(1, keepdim=True) + EPS)
    i = torch.arange(rows, device=DEV) // seg
    n = (n * W + B) * (1 + SC[i]) + SH[i]
    qkv = (n @ wqkv.double().T).view(rows, 3 * h, d)
    freq = 1e4 ** (-torch.arange(64, device=DEV, dtype=torch.float64) / 64)
    ang = torch.cat([pos.double()[:, :1] * freq, pos.double()[:, 1:] * freq], 1).repeat(rows // seg, 1)[:, None]
    t1, t2 = qkv[:, :2 * h, :128], qkv[:, :2 * h, 128:]
    qk = torch.cat([t1 * ang.cos() + t2 * ang.sin(), t2 * ang.cos() - t1 * ang.sin()], -1)
    qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS)
    outs = []
    for s in range(rows // seg):
        q, k, v = (t[s * seg:(s + 1) * seg].transpose(0, 1) for t in (qk[:, :h], qk[:, h:], qkv[:, 2 * h:]))
        outs.append((torch.softmax(q @ k.transpose(1, 2) * d ** -0.5, -1) @ v).transpose(0, 1))
    out = torch.cat(outs)
    ref = torch.autograd.grad((out * do.double()).sum(), leaves)
    tol = 12 * U
    rel = lambda a, r: ((a.double() - r).norm() / r.norm()).item()  # noqa: E731
    assert rel(saved[3], out) <= tol
    for name, g, r in zip(("dx", "dw", "db", "dshift", "dscale"), grads[1:], ref):
        assert rel(g, r) <= tol, name


def test_attention_branch_in_graphs_and_on_streams():
    """Two captured graphs (own workspaces each) replayed with new inputs, with eager work between the replays, and a
    run on another stream: all equal to the eager result, bit for bit."""
    args = [block_setup(seed) for seed in (0, 50)]

    def step(x, w, b, shift, scale, wqkv, pos, pairs, cu, h, d, do):
        saved = block(x, w, b, shift, scale, wqkv, pos, pairs, cu, h, d)
        return saved + block_bwd(do, x, w, b, scale, wqkv, pos, pairs, cu, h, d, *saved)

    expect = [step(*a) for a in args]
    graphs = []
    for a in args:
        step(*a)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(*a)
        graphs.append((g, res))
    for turn in range(3):
        for (g, _) in graphs:
            g.replay()
        junk = step(*args[turn % 2])  # eager work between replays
        torch.cuda.synchronize()
        for (_, res), exp in zip(graphs, expect):
            assert all(torch.equal(r, e) for r, e in zip(res, exp))
        assert all(torch.equal(r, e) for r, e in zip(junk, expect[turn % 2]))
        for _, res in graphs:
            for r in res:
                r.zero_()
    # new inputs in place
    for t, s in zip(args[0], args[1]):
        if torch.is_tensor(t):
            t.copy_(s)
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(r, e) for r, e in zip(graphs[0][1], expect[1]))
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(step(*args[1]))
    for s in side:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for res in got:
        assert all(torch.equal(r, e) for r, e in zip(res, expect[1]))


def test_offsets_past_32_bits():
    """Rows 2^22 elements apart, the last ones more than 2^31 elements behind the first: the results of packed rows."""
    rows, far = 600, 1 << 22
    buf = torch.empty(rows, far, device=DEV, dtype=BF)
    at = iter(range(0, far, 1024))

    def spread(like, fill=True):
        c, width = next(at), like[0].numel()
        v = buf[:, c:c + width].unflatten(1, like.shape[1:])
        return v.copy_(like) if fill else v

    q, k, v, do = attn_inputs(64, 2, 1, [rows], [rows], seed=70)
    cu, scale = cu_of([rows]), 64 ** -0.5
    out, lse = nat.attn_varlen_lse(q, k, v, cu, cu, scale)
    grads = nat.attn_varlen_bwd(do, q, k, v, out, lse, cu, cu, scale)
    Q, K, V, DO, O = spread(q), spread(k), spread(v), spread(do), spread(q, False)
    L = torch.empty_like(lse)
    nat.attn_varlen_lse(Q, K, V, cu, cu, scale, O, L)
    into = [spread(t, False) for t in (q, k, v)]
    nat.attn_varlen_bwd(DO, Q, K, V, O, L, cu, cu, scale, *into)
    assert torch.equal(O, out) and torch.equal(L, lse)
    assert all(torch.equal(a, b) for a, b in zip(into, grads))
    pos = torch.arange(2 * rows, device=DEV, dtype=torch.int32).view(rows, 2)
    y, r = nat.rope_axes(q, pos, (16, 16), norm=True)
    Y, R = nat.rope_axes(Q, pos, (16, 16), norm=True, out=spread(q, False))
    assert torch.equal(Y, y) and torch.equal(R, r)
    back = nat.rope_axes_bwd(DO, pos, (16, 16), y=Y, rstd=R, out=spread(q, False))
    assert torch.equal(back, nat.rope_axes_bwd(do, pos, (16, 16), y=y, rstd=r))
    x, w, b, shift, sc, dy = norm_inputs(rows, 640, 250, True, "rows", BF, False)
    x = x.contiguous()
    X, DY = spread(x), spread(dy)
    assert torch.equal(nat.layernorm_modulate(X, w, b, shift, sc, 250, out=spread(x, False)),
                       nat.layernorm_modulate(x, w, b, shift, sc, 250))
    got = nat.norm_modulate_bwd(DY, X, w, b, sc, 250, dx=spread(x, False))
    assert all(torch.equal(a, e) for a, e in zip(got, nat.norm_modulate_bwd(dy, x, w, b, sc, 250)))


def test_long_rows_and_many_sequences_in_a_graph():
    """What takes other launches than the branch above: norms of 8192 columns, and more than 64 sequences, whose work
    lists are made on the device; replayed with other lengths than captured."""
    x, w, b, shift, sc, dy = norm_inputs(6, 8192, 4, True, "rows", torch.float32, False)
    x = x.contiguous()
    ql, kl = [1, 9, 0, 4] * 20, [2, 0, 70, 5] * 20
    q, k, v, do = attn_inputs(64, 2, 2, ql, kl, seed=80)
    cq, ck = cu_of(ql), cu_of(kl)

    def run():
        y = nat.layernorm_modulate(x, w, b, shift, sc, 4)
        out, lse = nat.attn_varlen_lse(q, k, v, cq, ck, 0.125)
        return (y, *nat.norm_modulate_bwd(dy, x, w, b, sc, 4), out, lse,
                *nat.attn_varlen_bwd(do, q, k, v, out, lse, cq, ck, 0.125))

    run()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = run()
    for turn in range(3):
        if turn:
            cq.copy_(cu_of(ql[turn:] + ql[:turn]))
            ck.copy_(cu_of(kl[turn:] + kl[:turn]))
        for t in res:
            t.zero_()
        g.replay()
        expect = run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(res, expect))
