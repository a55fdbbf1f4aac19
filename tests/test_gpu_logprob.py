"""token_logprobs and topk_distillation_loss on a B200 against their definitions in 64 bits.

Tolerances, with u = 2^-24 (half a step of f32).  A row's sums are f32: a term 2^z carries the ex2's
2 ulp (4 u), and z = (x - m) c three roundings, 3 u |z|; a sum of n terms in a row adds n u, where n is
the longest chain: 8 within a unit, V / 2048 + 1 units per thread, and at most 64 roundings in the
merges (5 lanes + 7 warps, a few each; parts of a row add fewer).  So s is good to (n + 72) u plus
3 u E[|z|], and log p to that plus 6 u (|log p| + 1): z again, its fma and the product with ln 2.
The entropy adds t = sum p z: (n + 72) u E|z| + 3 u E[z^2].  A gradient is p times a factor, p good to
the error of log p plus 4 u, plus half a step of the output type.  All norms are taken per element."""
import collections

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


TokenRows = collections.namedtuple("TokenRows", "logprob entropy top_logprobs top_ids")


def chain(V):
    return V // 2048 + 1 + 72


def lp_tol(logp, V):
    """Of log p, from its 64-bit value."""
    p = logp.exp()
    ez = torch.where(p > 0, p * logp.abs(), 0.0).sum(-1, keepdim=True) + 1  # |z| ln 2 <= |log p| + log s <= ...
    return U * (chain(V) + 4 * ez + 6 * (torch.where(torch.isinf(logp), 0.0, logp.abs()) + 1))


def ent_tol(logp, V):
    p = logp.exp()
    l = torch.where(p > 0, logp.abs(), 0.0)
    m1, m2 = (p * l).sum(-1), (p * l * l).sum(-1)
    return U * ((chain(V) + 8) * (1 + 2 * m1) + 8 * (m2 + m1 + 1))


def top_ref(x, k):
    """Columns of the k largest, NaN first, ties to the lowest column."""
    x = x.detach().cpu().double().numpy().reshape(-1, x.shape[-1])
    out = np.empty((x.shape[0], k), np.int64)
    cols = np.arange(x.shape[1])
    for r in range(x.shape[0]):
        v = np.where(np.isnan(x[r]), 0.0, x[r]) + 0.0
        out[r] = np.lexsort((cols, -v, ~np.isnan(x[r])))[:k]
    return out


def make(cuda, rows, V, dtype, seed, scale=2.5):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = (torch.randn((rows, V), generator=g, device=cuda) * scale).to(dtype)
    tok = torch.randint(0, V, (rows,), generator=g, device=cuda)
    return x, tok, g


def check_score(x, tok, out, T, k, mask=None):
    V = x.shape[-1]
    x2, tok2 = x.reshape(-1, V), tok.reshape(-1)
    logp = torch.log_softmax(x2.double() / T, -1)
    keep = torch.ones(x2.shape[0], dtype=torch.bool, device=x.device) if mask is None else mask.reshape(-1) != 0
    tol = lp_tol(logp, V)
    ref = logp.gather(1, tok2[:, None].long() % V)[:, 0]
    err = (out.logprob.reshape(-1).double() - torch.where(keep, ref, 0.0)).abs()
    same_inf = torch.isinf(ref) & keep
    assert torch.equal(torch.isinf(out.logprob.reshape(-1)), same_inf)
    assert (err[~same_inf] <= tol.gather(1, tok2[:, None].long() % V)[:, 0][~same_inf]).all()
    if out.entropy is not None:
        p = logp.exp()
        H = -torch.where(p > 0, p * logp, 0.0).sum(-1)
        eerr = (out.entropy.reshape(-1).double() - torch.where(keep, H, 0.0)).abs()
        assert (eerr <= ent_tol(logp, V)).all(), (eerr / ent_tol(logp, V)).max()
    if k:
        ids = torch.from_numpy(top_ref(x2, k)).to(x.device)
        got = out.top_ids.reshape(-1, k)
        assert torch.equal(got, torch.where(keep[:, None], ids, -1))
        tref, ttol = logp.gather(1, ids), tol.gather(1, ids)
        glp = out.top_logprobs.reshape(-1, k).double()
        assert (glp[~keep] == float("-inf")).all()
        fin = keep[:, None] & ~torch.isinf(tref)
        assert torch.equal(torch.isinf(glp) & keep[:, None], torch.isinf(tref) & keep[:, None])
        assert ((glp - tref).abs()[fin] <= ttol[fin]).all()


SIZES = [(1, 1), (3, 2), (2, 7), (5, 31), (4, 255), (3, 2047), (2, 2048), (2, 2049), (3, 8191), (2, 8193), (7, 16391),
         (3, 50257), (2, 128256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V", SIZES)
def test_score_sizes(cuda, rows, V, dtype):
    from macrogpt_jax_b200.logprobs import token_logprobs
    x, tok, _ = make(cuda, rows, V, dtype, rows * 1000 + V)
    for k, T in ((0, 1.0), (min(V, 1), 0.7), (min(V, 20), 2.0), (min(V, 256), 1.0)):
        check_score(x, tok, token_logprobs(x, tok, top_k=k, temperature=T), T, k)


@pytest.mark.parametrize("rows", [1, 2, 3, 9, 40, 75, 150, 300, 700])
def test_score_row_counts(cuda, rows):
    """Every number of parts that a row is split into."""
    from macrogpt_jax_b200.logprobs import token_logprobs
    for V in (5000, 70001):
        x, tok, _ = make(cuda, rows, V, torch.bfloat16, rows)
        check_score(x, tok, token_logprobs(x, tok, top_k=33), 1.0, 33)


@pytest.mark.parametrize("rows,V,dtype", [(900, 115001, torch.bfloat16), (1000, 70001, torch.bfloat16),
                                          (900, 60001, torch.float32), (2000, 8192, torch.bfloat16),
                                          (2000, 20001, torch.float32), (1200, 33001, torch.bfloat16),
                                          (420, 300001, torch.bfloat16), (800, 270001, torch.bfloat16)])
def test_score_many_rows(cuda, rows, V, dtype):
    """The choices of CTA size and parts for many rows (row starts at every alignment)."""
    from macrogpt_jax_b200.distill import topk_distillation_loss
    from macrogpt_jax_b200.logprobs import token_logprobs
    x, tok, g = make(cuda, rows, V, dtype, rows)
    some = torch.randperm(rows, generator=g, device=cuda)[:150]
    for k in (0, 20, 100):
        out = token_logprobs(x, tok, top_k=k)
        check_score(x[some], tok[some], TokenRows(*(None if t is None else t[some] for t in out)), 1.0, k)
    ids = torch.randint(0, V, (rows, 40), generator=g, device=cuda)
    t = torch.randn((rows, 40), generator=g, device=cuda)
    loss = topk_distillation_loss(x, ids, t)[some]
    rl, ltol, *_ = distill_ref(x[some], ids[some], t[some], 1.0)
    assert ((loss.double() - rl).abs() <= ltol).all()


@pytest.mark.parametrize("k", [1, 2, 3, 4, 5, 8, 9, 16, 17, 64, 65, 128, 129, 255, 256])
def test_top_k_values(cuda, k):
    from macrogpt_jax_b200.logprobs import token_logprobs
    x, tok, _ = make(cuda, 6, 33333, torch.bfloat16, k)
    check_score(x, tok, token_logprobs(x, tok, top_k=k), 1.0, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 300])
def test_top_orders(cuda, dtype, rows):
    """Rows that fill the candidate buffer or tie: constant, rising, falling, two values, one peak, many
    equal maxima at the end, zeros of both signs, a prefix or all but a few columns of -inf."""
    from macrogpt_jax_b200.logprobs import token_logprobs
    V = 40000
    ramp = torch.arange(V, device=cuda, dtype=torch.float32) / 1024 - 20
    g = torch.Generator(device=cuda).manual_seed(1)
    rnd = torch.randn(V, generator=g, device=cuda)
    kinds = [torch.zeros(V, device=cuda), ramp, ramp.flip(0), (torch.arange(V, device=cuda) % 2).float(),
             torch.where(torch.arange(V, device=cuda) == V - 1, 5.0, 0.0),
             torch.where(torch.arange(V, device=cuda) >= V - 400, 3.0, rnd),
             torch.where(rnd > 0, 0.0, -0.0), torch.where(torch.arange(V, device=cuda) < V - 7, float("-inf"), rnd),
             torch.where(torch.arange(V, device=cuda) % 9001 == 3, rnd, float("-inf")),
             torch.full((V,), torch.finfo(dtype).min, device=cuda),
             torch.where(rnd > 2, rnd, torch.tensor(torch.finfo(dtype).min, device=cuda))]
    base = torch.stack(kinds).to(dtype)
    x = base.repeat(-(-rows // len(kinds)) if rows > 1 else 1, 1)
    for i in (range(len(kinds)) if rows == 1 else [None]):
        xi = x if i is None else x[i:i + 1]
        tok = torch.full((xi.shape[0],), V - 1, device=cuda)
        for k in (1, 20, 200):
            check_score(xi, tok, token_logprobs(xi, tok, top_k=k), 1.0, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("scale,T", [(1e30, 0.5), (1e-30, 1.0), (2.5, 0.01), (2.5, 1e4), (40.0, 1.0)])
def test_score_magnitudes(cuda, dtype, scale, T):
    """Logits so large that the others have no weight, so small that all have the same, and temperatures
    that do either."""
    from macrogpt_jax_b200.logprobs import token_logprobs
    x, tok, _ = make(cuda, 9, 12345, dtype, 31, scale)
    check_score(x, tok, token_logprobs(x, tok, top_k=11, temperature=T), T, 11)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [3, 210, 700])
@pytest.mark.parametrize("count", [900, 1300, 2600])
def test_top_ties_in_one_warp(cuda, dtype, rows, count):
    """More equal maxima than the gathered keys hold, all of them in columns that one warp of a CTA reads:
    the search of the whole row then leaves few keys, in one warp's list."""
    from macrogpt_jax_b200.logprobs import token_logprobs
    V = 50000 if rows < 700 else 20000
    per = 8 if dtype == torch.bfloat16 else 4
    threads = 256 if rows < 592 else 128
    col = torch.arange(V, device=cuda)
    warp0 = col // per % threads < 32
    g = torch.Generator(device=cuda).manual_seed(rows + count)
    x = torch.randn((rows, V), generator=g, device=cuda)
    x[:, col[warp0][:count]] = 9.0
    x = x.to(dtype)
    tok = torch.randint(0, V, (rows,), generator=g, device=cuda)
    for k in (1, 7, 100):
        check_score(x[:3], tok[:3], take(token_logprobs(x, tok, top_k=k), slice(0, 3)), 1.0, k)


def take(out, rows):
    return type(out)(*(t[rows] for t in out))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_score_not_finite(cuda, dtype):
    """+inf, NaN and rows of only -inf give NaN, and only in their own row; the order stays defined."""
    from macrogpt_jax_b200.logprobs import token_logprobs
    x, tok, _ = make(cuda, 6, 9000, dtype, 3)
    x[1, 77] = float("nan")
    x[2, 5] = float("inf")
    x[3] = float("-inf")
    x[4, 8500:] = float("nan")
    out = token_logprobs(x, tok, top_k=30)
    for t in (out.logprob, out.entropy):
        assert torch.equal(torch.isnan(t), torch.tensor([0, 1, 1, 1, 1, 0], device=cuda).bool())
    assert torch.equal(out.top_ids, torch.from_numpy(top_ref(x, 30)).to(cuda))
    good = torch.tensor([0, 5], device=cuda)
    check_score(x[good], tok[good], take(out, good), 1.0, 30)


def test_score_tokens_and_mask(cuda):
    """int32 and int64 tokens, tokens from the end, tokens without a column; every mask type, a mask
    that leaves nothing, masked rows of NaN."""
    from macrogpt_jax_b200.logprobs import token_logprobs
    x, tok, g = make(cuda, 40, 3001, torch.bfloat16, 8)
    a = token_logprobs(x, tok, top_k=4)
    b = token_logprobs(x, (tok - 3001).to(torch.int32), top_k=4)
    c = token_logprobs(x, tok.to(torch.int16))
    assert torch.equal(a.logprob, b.logprob) and torch.equal(a.logprob, c.logprob)
    odd = tok.clone()
    odd[3], odd[4] = 3001, -3002
    assert torch.isnan(token_logprobs(x, odd).logprob).nonzero().flatten().tolist() == [3, 4]
    keep = torch.rand(40, generator=g, device=cuda) > 0.4
    x[~keep] = float("nan")
    for m in (keep, keep.to(torch.uint8) * 3, keep.int() * -1, keep.long()):
        check_score(torch.nan_to_num(x), tok, token_logprobs(x, tok, top_k=4, mask=m), 1.0, 4, keep)
    none = token_logprobs(x, tok, top_k=4, mask=torch.zeros(40, dtype=torch.bool, device=cuda))
    assert (none.logprob == 0).all() and (none.entropy == 0).all() and (none.top_ids == -1).all()
    only = token_logprobs(x, None, top_k=4, entropy=False, mask=keep)
    assert only.logprob is None and only.entropy is None
    assert torch.equal(only.top_ids, token_logprobs(x, tok, top_k=4, mask=keep).top_ids)


def views(cuda, dtype):
    g = torch.Generator(device=cuda).manual_seed(5)
    big = (torch.randn((3, 6, 1207), generator=g, device=cuda) * 3).to(dtype)
    return {"shift": big[:, :-1], "tail": big[:, 1:], "columns": big[..., 3:1100], "head": big[..., :1200],
            "steps": big[:, ::2], "swap": big.transpose(0, 1), "one": big[1, 2], "expanded": big[:1].expand(4, 6, 1207),
            "levels": big.reshape(3, 2, 3, 1207)[:, :1, :2], "column_steps": big[..., ::2]}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["shift", "tail", "columns", "head", "steps", "swap", "one", "expanded", "levels",
                                  "column_steps"])
def test_strides(cuda, dtype, kind):
    """Views give what their contiguous copies give, forward and backward: the same columns, and numbers
    that are both within their tolerance of the definition's.  (Not the same bits: a row's sums are
    grouped from its first 16-byte boundary on, so another alignment adds in another order.)"""
    from macrogpt_jax_b200.distill import topk_distillation_loss
    from macrogpt_jax_b200.logprobs import TokenLogprobs, token_logprobs
    x = views(cuda, dtype)[kind].detach()
    y = x.clone(memory_format=torch.contiguous_format)
    lead, V = x.shape[:-1], x.shape[-1]
    tok = torch.arange(max(1, x[..., 0].numel()), device=cuda).reshape(lead) * 37 % V
    ids = (tok[..., None] + torch.arange(5, device=cuda) * 11) % V
    teacher = torch.linspace(2, 0, 5, device=cuda).expand(*lead, 5)
    res = []
    for t in (x, y):
        t = t.requires_grad_(True)
        out = token_logprobs(t, tok, top_k=7, temperature=0.9)
        loss = topk_distillation_loss(t, ids, teacher, temperature=1.3)
        g1, = torch.autograd.grad((out.logprob.sum() + out.entropy.sum() + out.top_logprobs.sum()), t)
        g2, = torch.autograd.grad(loss.sum(), t)
        assert g1.shape == t.shape and g2.shape == t.shape
        res.append((*out, loss, g1, g2))
    for a, b in zip(*res):
        assert a.shape == b.shape and a.dtype == b.dtype
    assert torch.equal(res[0][3], res[1][3])
    x2 = y.reshape(-1, V)
    n = x2.shape[0]
    ones = torch.ones(n, device=cuda)
    for out in res:
        lp, ent, top_lp, top_id, loss, g1, g2 = (v.detach() for v in out)
        check_score(y, tok, TokenLogprobs(lp, ent, top_lp, top_id), 0.9, 7)
        rl, ltol, rg, gtol, _ = distill_ref(x2, ids.reshape(n, 5), teacher.reshape(n, 5), 1.3)
        assert ((loss.reshape(-1).double() - rl).abs() <= ltol).all()
        check_grad(g2.reshape(n, V), rg, gtol)
        check_grad(g1.reshape(n, V), *grad_ref(x2, tok.reshape(-1), 0.9, ones, ones, torch.ones((n, 7), device=cuda),
                                               top_id.reshape(n, 7)))


def grad_ref(x, tok, T, dlp, dent, dtop, ids):
    """(gradient, tolerance before the output's rounding) in 64 bits."""
    V = x.shape[-1]
    logp = torch.log_softmax(x.double() / T, -1)
    p = logp.exp()
    safe = torch.where(p > 0, logp, 0.0)
    H = -(p * safe).sum(-1, keepdim=True)
    w = torch.zeros_like(p)
    wabs = torch.zeros_like(p)
    G = torch.zeros(x.shape[0], 1, dtype=torch.float64, device=x.device)
    Gabs = G.clone()
    for g, cols in ((dlp, tok[:, None]), (dtop, ids)):
        if g is not None:
            g = g.double().reshape(x.shape[0], -1)
            w.scatter_add_(1, cols, g)
            wabs.scatter_add_(1, cols, g.abs())
            G = G + g.sum(1, keepdim=True)
            Gabs = Gabs + g.abs().sum(1, keepdim=True) * (1 + g.shape[1])
    h = torch.zeros_like(G) if dent is None else dent.double()[:, None]
    grad = (w - p * (G + h * (safe + H))) / T
    rel = lp_tol(logp, V) + 8 * U
    tol = (wabs * 4 * U + p * (Gabs * (rel + 8 * U) + h.abs() * (rel * (safe.abs() + H + 1) + ent_tol(logp, V)[:, None]
                                                                 + 8 * U * (safe.abs() + H)))) / T
    return grad, tol


def check_grad(got, ref, tol):
    half = torch.finfo(got.dtype).eps / 2
    err = (got.double() - ref).abs()
    bound = tol * (1 + half) + half * ref.abs() + torch.finfo(got.dtype).tiny
    assert (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 7), (4, 2049), (6, 8193), (3, 50257), (2, 128256), (300, 4999)])
def test_score_gradient(cuda, dtype, rows, V):
    from macrogpt_jax_b200.logprobs import token_logprobs
    x, tok, g = make(cuda, rows, V, dtype, V + 1)
    x = x.requires_grad_(True)
    k = min(V, 12)
    for T, kk in ((1.0, 0), (0.6, k), (1.7, k)):
        out = token_logprobs(x, tok, top_k=kk, temperature=T)
        dlp, dent = (torch.randn(rows, generator=g, device=cuda) for _ in range(2))
        dtop = torch.randn((rows, kk), generator=g, device=cuda) if kk else None
        for parts in ("l", "e", "le") + (("t", "let") if kk else ()):
            outs = [(out.logprob, dlp, "l"), (out.entropy, dent, "e"), (out.top_logprobs, dtop, "t")]
            use = [(o, d) for o, d, n in outs if n in parts]
            got, = torch.autograd.grad([o for o, _ in use], x, [d for _, d in use], retain_graph=True)
            ref, tol = grad_ref(x.detach(), tok, T, dlp if "l" in parts else None, dent if "e" in parts else None,
                                dtop if "t" in parts else None, out.top_ids if kk else None)
            check_grad(got, ref, tol)


def test_score_gradient_masks_and_infinities(cuda):
    """Masked rows: gradient 0 even where they hold NaN; columns of -inf: 0; a token without a column:
    only the dense part; .sum() and .mean() send one value for all rows."""
    from macrogpt_jax_b200.logprobs import token_logprobs
    x, tok, g = make(cuda, 24, 5003, torch.float32, 2)
    keep = torch.rand(24, generator=g, device=cuda) > 0.5
    x[:, ::7] = float("-inf")
    clean = x.clone()
    x[~keep] = float("nan")
    tok = torch.where(tok % 7 == 0, tok + 1, tok) % 5003
    x = x.requires_grad_(True)
    out = token_logprobs(x, tok, top_k=3, mask=keep)
    got, = torch.autograd.grad(out.logprob.sum() + 0.5 * out.entropy.mean(), x)
    ref, tol = grad_ref(clean, tok, 1.0, torch.ones(24, device=cuda), torch.full((24,), 0.5 / 24, device=cuda), None,
                        None)
    check_grad(got[keep], ref[keep], tol[keep])
    assert (got[~keep] == 0).all() and (got[:, ::7] == 0).all()
    bad = tok.clone()
    bad[keep.nonzero()[0]] = 5003
    y = clean.clone().requires_grad_(True)
    got, = torch.autograd.grad(token_logprobs(y, bad).logprob, y, torch.ones(24, device=cuda))
    r = int(keep.nonzero()[0])
    p = torch.softmax(clean[r].double(), -1)
    assert (got[r].double() + p).abs().max() <= 200 * U


def test_masked_rows_ignore_their_upstream_gradient(cuda):
    """A masked row's gradient is 0 whatever comes back for it, NaN included."""
    from macrogpt_jax_b200.distill import topk_distillation_loss
    from macrogpt_jax_b200.logprobs import token_logprobs
    x, tok, _ = make(cuda, 6, 4001, torch.bfloat16, 17)
    keep = torch.tensor([1, 0, 1, 0, 0, 1], device=cuda).bool()
    d = torch.where(keep, 1.0, float("nan"))
    x = x.requires_grad_(True)
    out = token_logprobs(x, tok, top_k=2, mask=keep)
    loss = topk_distillation_loss(x, out.top_ids, out.top_logprobs.detach(), mask=keep)
    for o, u in ((out.logprob, d), (out.entropy, d), (out.top_logprobs, d[:, None].expand(6, 2)), (loss, d)):
        got, = torch.autograd.grad(o, x, u, retain_graph=True)
        assert got[keep].isfinite().all() and got[keep].any() and (got[~keep] == 0).all()


def test_score_gradient_by_differences(cuda):
    """The formula's gradient against central differences of the operator itself (f32, one row)."""
    from macrogpt_jax_b200.logprobs import token_logprobs
    V, T, eps = 9, 0.8, 2.0 ** -6
    x, _, g = make(cuda, 1, V, torch.float32, 4, 1.0)
    tok = torch.tensor([4], device=cuda)

    def f(t):
        o = token_logprobs(t, tok.expand(t.shape[0]), top_k=2, temperature=T)
        return 1.5 * o.logprob[..., None] - 0.7 * o.entropy[..., None] + o.top_logprobs[..., 1:2]

    xg = x.clone().requires_grad_(True)
    got, = torch.autograd.grad(f(xg).sum(), xg)
    pts = torch.cat([x + eps * torch.eye(V, device=cuda), x - eps * torch.eye(V, device=cuda)])
    val = f(pts).double()[:, 0]
    num = (val[:V] - val[V:]) / (2 * eps)
    # rounding: values below 16 good to 100 u each; curvature: third derivatives below 40 / T^3
    assert (got[0].double() - num).abs().max() <= 2 * 16 * 100 * U / (2 * eps) + 40 / T ** 3 * eps ** 2 / 6


def distill_ref(x, ids, t, T, keep=None):
    V = x.shape[-1]
    logp = torch.log_softmax(x.double() / T, -1)
    has = (ids >= 0) & (ids < V)
    tt = (t.double() / T).masked_fill(ids < 0, float("-inf"))
    live = ~torch.isinf(tt).all(-1, keepdim=True)
    q = torch.where(live, torch.softmax(torch.where(live, tt, 0.0), -1), 0.0)
    lq = torch.where(q > 0, q.log(), 0.0)
    lp = logp.gather(1, ids.clamp(0, V - 1).long())
    loss = torch.where(q > 0, q * (lq - lp), 0.0).sum(-1)
    dense = torch.zeros_like(logp).scatter_add_(1, ids.clamp(0, V - 1).long(), torch.where(has, q, 0.0))
    grad = (logp.exp() * live - dense) / T
    K = ids.shape[1]
    tl = lp_tol(logp, V).gather(1, ids.clamp(0, V - 1).long())
    qerr = U * (K + 16 + 8 * lq.abs())  # relative, of q; absolute, of log q
    fin = torch.where(q > 0, (lq - lp).abs(), 0.0)
    ltol = (q * (qerr * (fin + 1) + tl + (K + 8) * U * fin)).sum(-1) + 4 * U * loss.abs()
    qd = torch.zeros_like(logp).scatter_add_(1, ids.clamp(0, V - 1).long(), q * (qerr + K * U + 8 * U))
    gtol = (logp.exp() * (lp_tol(logp, V) + 16 * U) + qd) / T
    return loss, ltol, grad, gtol, live[:, 0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V,K", [(1, 1, 1), (2, 5, 5), (5, 300, 17), (3, 2049, 64), (4, 8193, 100),
                                      (3, 50257, 1), (2, 128256, 1024), (300, 5001, 32), (7, 4096, 0)])
def test_distill(cuda, dtype, rows, V, K):
    from macrogpt_jax_b200.distill import topk_distillation_loss
    x, _, g = make(cuda, rows, V, dtype, V + K)
    x = x.requires_grad_(True)
    ids = torch.rand((rows, V), generator=g, device=cuda).argsort(-1)[:, :K] if K <= V else None
    t = (torch.randn((rows, K), generator=g, device=cuda) * 2).to(dtype)
    d = torch.randn(rows, generator=g, device=cuda)
    for T, idt in ((1.0, torch.int64), (2.0, torch.int32)):
        loss = topk_distillation_loss(x, ids.to(idt), t, temperature=T)
        rl, ltol, rg, gtol, _ = distill_ref(x.detach(), ids, t, T)
        assert ((loss.double() - rl).abs() <= ltol).all(), ((loss.double() - rl).abs() / ltol).max()
        got, = torch.autograd.grad(loss, x, d)
        w = d.double()[:, None]
        check_grad(got, rg * w, gtol * w.abs() + 4 * U * (rg * w).abs())


def test_distill_rows(cuda):
    """Absent entries, rows without entries, weights of zero, columns given twice, ids without a column,
    banned student columns, masked rows of NaN."""
    from macrogpt_jax_b200.distill import topk_distillation_loss
    V, K = 10007, 12
    x, _, g = make(cuda, 10, V, torch.float32, 11)
    ids = torch.rand((10, V), generator=g, device=cuda).argsort(-1)[:, :K]
    t = torch.randn((10, K), generator=g, device=cuda)
    ids[0, 5:] = -1
    ids[1] = -1
    t[2, :6] = float("-inf")
    t[3] = float("-inf")
    ids[4, 3] = ids[4, 9] = ids[4, 0]          # one column three times
    x[6, ids[6, 1:]] = float("-inf")
    t[6, 1:] = float("-inf")                   # banned columns without weight
    keep = torch.ones(10, dtype=torch.bool, device=cuda)
    keep[7] = False
    clean = x.clone()
    x[7] = float("nan")
    x = x.requires_grad_(True)
    loss = topk_distillation_loss(x, ids, t, mask=keep)
    got, = torch.autograd.grad(loss, x, torch.ones(10, device=cuda))
    rl, ltol, rg, gtol, live = distill_ref(clean, ids, t, 1.0)
    assert live.tolist() == [True, False, True, False] + [True] * 6
    rl, rg = torch.where(keep, rl, 0.0), torch.where(keep[:, None], rg, 0.0)
    assert ((loss.double() - rl).abs() <= ltol).all()
    check_grad(got, rg, gtol)
    for r in (1, 3, 7):
        assert loss[r] == 0 and (got[r] == 0).all()
    # an id past the last column: NaN, a banned column with weight: +inf; both leave other rows alone
    ids2, y = ids.clone(), clean.clone()
    ids2[8, 2] = V
    y[9, ids[9, 0]] = float("-inf")
    loss2 = topk_distillation_loss(y, ids2, t)
    assert torch.isnan(loss2[8]) and loss2[9] == float("inf")
    assert torch.equal(loss2[:7], topk_distillation_loss(clean, ids, t)[:7])


def test_distill_gradient_by_differences(cuda):
    from macrogpt_jax_b200.distill import topk_distillation_loss
    V, T, eps = 11, 1.5, 2.0 ** -6
    x, _, g = make(cuda, 1, V, torch.float32, 6, 1.0)
    ids = torch.tensor([[3, 7, 3, 10]], device=cuda)
    t = torch.tensor([[1.0, 0.2, -0.5, 0.1]], device=cuda)
    f = lambda y: topk_distillation_loss(y, ids.expand(len(y), 4), t.expand(len(y), 4), temperature=T)  # noqa: E731
    xg = x.clone().requires_grad_(True)
    got, = torch.autograd.grad(f(xg).sum(), xg)
    pts = torch.cat([x + eps * torch.eye(V, device=cuda), x - eps * torch.eye(V, device=cuda)])
    val = f(pts).double()
    num = (val[:V] - val[V:]) / (2 * eps)
    assert (got[0].double() - num).abs().max() <= 2 * 16 * 100 * U / (2 * eps) + 10 / T ** 3 * eps ** 2 / 6


def test_distill_from_itself_is_zero(cuda):
    """Teacher entries over the whole vocabulary equal to the student's logits: loss and gradient are
    rounding only."""
    from macrogpt_jax_b200.distill import topk_distillation_loss
    from macrogpt_jax_b200.logprobs import token_logprobs
    x, _, _ = make(cuda, 5, 256, torch.float32, 9)
    top = token_logprobs(x, None, top_k=256, entropy=False)
    x = x.requires_grad_(True)
    loss = topk_distillation_loss(x, top.top_ids, top.top_logprobs)
    got, = torch.autograd.grad(loss.sum(), x)
    _, ltol, _, gtol, _ = distill_ref(x.detach(), top.top_ids, top.top_logprobs, 1.0)
    # the teacher's values carry the error of a log probability themselves
    p = torch.softmax(x.detach().double(), -1)
    own = lp_tol(torch.log_softmax(x.detach().double(), -1), 256)
    assert (loss.double().abs() <= ltol + 2 * own.amax(-1)).all()
    assert (got.double().abs() <= gtol + p * 2 * own.amax(-1, keepdim=True)).all()


def test_teacher_to_student(cuda):
    """A run of them together: the teacher's top entries, the student's distillation step, the log
    probabilities of the labels, one backward pass over the sum."""
    from macrogpt_jax_b200.distill import topk_distillation_loss
    from macrogpt_jax_b200.logprobs import token_logprobs
    from macrogpt_jax_b200.next_token_loss import ntp_args
    b, n, V = 3, 17, 4099
    g = torch.Generator(device=cuda).manual_seed(12)
    inputs = torch.randint(0, V, (b, n), generator=g, device=cuda)
    inputs[1, 9:] = 0
    targets, mask = ntp_args(inputs, pad_token_id=0)
    tl = (torch.randn((b, n, V), generator=g, device=cuda) * 3).bfloat16()
    sl = (torch.randn((b, n, V), generator=g, device=cuda) * 3).bfloat16().requires_grad_(True)
    with torch.no_grad():
        top = token_logprobs(tl, None, top_k=16, temperature=1.0, mask=mask, entropy=False)
    loss = topk_distillation_loss(sl, top.top_ids, top.top_logprobs, temperature=2.0, mask=mask)
    lp = token_logprobs(sl, targets, mask=mask, entropy=False).logprob
    total = 4.0 * loss.sum() - lp.sum()
    got, = torch.autograd.grad(total, sl)
    x = sl.detach().reshape(-1, V)
    keep = mask.reshape(-1) != 0
    rl, ltol, rg, gtol, _ = distill_ref(x, top.top_ids.reshape(-1, 16).clamp(min=-1), torch.where(
        keep[:, None], top.top_logprobs.reshape(-1, 16), 0.0), 2.0)
    assert ((loss.reshape(-1).double() - rl)[keep].abs() <= ltol[keep]).all() and (loss.reshape(-1)[~keep] == 0).all()
    g2, t2 = grad_ref(x, targets.reshape(-1), 1.0, -torch.ones(b * n, device=cuda), None, None, None)
    ref = torch.where(keep[:, None], 4 * rg + g2, 0.0)
    # two bf16 gradients and their bf16 sum: half a step of each
    half = torch.finfo(torch.bfloat16).eps / 2
    bound = 4 * gtol + t2 + half * ((4 * rg).abs() + g2.abs()) * (1 + half) + half * ref.abs() + 1e-30
    err = (got.reshape(-1, V).double() - ref).abs()
    assert (err[keep] <= bound[keep]).all() and (got.reshape(-1, V)[~keep] == 0).all()


def test_results_do_not_depend_on_the_run(cuda):
    """Same bits twice, on another stream, and replayed from a CUDA graph with new inputs."""
    from macrogpt_jax_b200.distill import topk_distillation_loss
    from macrogpt_jax_b200.graphs import GraphedStep
    from macrogpt_jax_b200.logprobs import token_logprobs
    x, tok, g = make(cuda, 37, 20011, torch.bfloat16, 21)
    ids = torch.rand((37, 20011), generator=g, device=cuda).argsort(-1)[:, :9]
    t = torch.randn((37, 9), generator=g, device=cuda)

    def step(x, tok, ids, t):
        x = x.detach().requires_grad_(True)
        out = token_logprobs(x, tok, top_k=50, temperature=0.9)
        loss = topk_distillation_loss(x, ids, t)
        g1, = torch.autograd.grad((out.logprob, out.entropy), x, (loss.detach(), loss.detach()))
        g2, = torch.autograd.grad(loss, x, out.logprob.detach())
        return tuple(v.detach() for v in (*out, loss, g1, g2))

    first = step(x, tok, ids, t)
    for a, b in zip(first, step(x, tok, ids, t)):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(x, tok, ids, t)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, other):
        assert torch.equal(a, b)
    graphed = GraphedStep(step, torch.zeros_like(x), torch.zeros_like(tok), torch.zeros_like(ids), torch.zeros_like(t))
    for _ in range(2):
        for a, b in zip(first, graphed(x, tok, ids, t)):
            assert torch.equal(a, b)


def test_no_rows(cuda):
    from macrogpt_jax_b200.distill import topk_distillation_loss
    from macrogpt_jax_b200.logprobs import token_logprobs
    x = torch.empty((2, 0, 9), device=cuda, requires_grad=True)
    out = token_logprobs(x, torch.empty((2, 0), dtype=torch.int64, device=cuda), top_k=3)
    assert out.logprob.shape == (2, 0) and out.top_ids.shape == (2, 0, 3)
    loss = topk_distillation_loss(x, torch.empty((2, 0, 4), dtype=torch.int64, device=cuda),
                                  torch.empty((2, 0, 4), device=cuda))
    (loss.sum() + out.logprob.sum()).backward()
    assert x.grad.shape == x.shape


def test_long_rows_past_32_bits(cuda):
    """Elements past 2^31: the last of 17000 rows of 128256 columns."""
    from macrogpt_jax_b200.logprobs import token_logprobs
    rows, V = 17000, 128256
    x = torch.zeros((rows, V), dtype=torch.bfloat16, device=cuda)
    x[-1, 1000:1010] = torch.arange(10, 20, device=cuda, dtype=torch.bfloat16)
    tok = torch.full((rows,), 1009, device=cuda)
    mask = torch.zeros(rows, dtype=torch.bool, device=cuda)
    mask[-2:] = True
    x = x.requires_grad_(True)
    out = token_logprobs(x, tok, top_k=3, mask=mask)
    assert out.top_ids[-1].tolist() == [1009, 1008, 1007] and out.top_ids[-2].tolist() == [0, 1, 2]
    got, = torch.autograd.grad(out.logprob.sum(), x)
    ref, tol = grad_ref(x.detach()[-2:], tok[-2:], 1.0, torch.ones(2, device=cuda), None, None, None)
    check_grad(got[-2:], ref, tol)
    assert not got[:5].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_ids_without_a_column(cuda, dtype):
    """A token outside [-V, V) and a teacher id >= V make their row's result NaN; the gradients leave them out
    and stay finite, in that row and in all others."""
    from macrogpt_jax_b200.distill import topk_distillation_loss
    from macrogpt_jax_b200.logprobs import token_logprobs
    V = 5001
    x, tok, g = make(cuda, 8, V, dtype, 23)
    tok[2], tok[5] = V, -V - 1
    x = x.requires_grad_(True)
    out = token_logprobs(x, tok, top_k=3)
    assert torch.isnan(out.logprob).nonzero().flatten().tolist() == [2, 5]
    assert out.entropy.isfinite().all() and out.top_logprobs.isfinite().all()
    got, = torch.autograd.grad(out.logprob, x, torch.ones(8, device=cuda))
    logp = torch.log_softmax(x.detach().double(), -1)
    inside = (tok >= 0) & (tok < V)
    ref = torch.zeros_like(logp).scatter_(1, tok.clamp(0, V - 1)[:, None], inside.double()[:, None]) - logp.exp()
    check_grad(got, ref, logp.exp() * (lp_tol(logp, V) + 16 * U) + 4 * U * ref.abs())
    ids = torch.rand((8, V), generator=g, device=cuda).argsort(-1)[:, :70]
    t = torch.randn((8, 70), generator=g, device=cuda)
    for row, j in ((1, 0), (4, 33), (6, 69)):
        ids[row, j] = (V, V + 7, 2 ** 31 - 1)[row // 3]
    for idt in (torch.int64, torch.int32):
        loss = topk_distillation_loss(x, ids.to(idt), t, temperature=1.5)
        assert torch.isnan(loss).nonzero().flatten().tolist() == [1, 4, 6]
        got, = torch.autograd.grad(loss, x, torch.ones(8, device=cuda))
        _, _, rg, gtol, _ = distill_ref(x.detach(), ids, t, 1.5)
        check_grad(got, rg, gtol)
