"""GPU tests of the token-model operators against their float64 definitions (token_reference.py, which also derives
every tolerance), at the sizes, masks and layouts where they can go wrong."""
import numpy as np
import pytest

import token_reference as ref
import zigneuron_b200 as zn

pytestmark = pytest.mark.gpu
NINF = -np.inf
I32, U32, F32 = np.int32, np.uint32, np.float32
GUARD = F32(-777.25)


@pytest.fixture(scope="module")
def be():
    b = zn.Backend(0)
    yield b
    b.deinit()


def zipf_tokens(rng, rows, vocab, pad=0.05):
    t = np.minimum((np.exp(rng.random(rows) * np.log(vocab + 1)) - 1).astype(np.int64), vocab - 1)
    t[rng.random(rows) < pad] = -1
    return t.astype(I32)


def padded(rng, rows, vocab, ld, scale=3.0):
    buf = np.full((rows, ld), GUARD, F32)
    buf[:, :vocab] = rng.standard_normal((rows, vocab)) * scale
    return buf


def free(*tensors):
    for t in tensors:
        t.free()


# ---- embedding -------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,vocab,dim", [(1, 1, 1), (1, 9, 4), (3, 7, 5), (33, 100, 64), (257, 1000, 129), (1000, 50, 260),
                                            (4099, 3001, 96), (2, 11, 4100), (20000, 17, 8)])
def test_embedding_forward(be, rows, vocab, dim):
    rng = np.random.default_rng(rows + dim)
    table = rng.standard_normal((vocab, dim)).astype(F32)
    tok = rng.integers(-1, vocab, rows).astype(I32)
    want = ref.embedding_forward(table, tok, 0.3)
    out = np.full((rows, dim), GUARD, F32)
    be.embeddingForward(table, tok, out, rows, vocab, dim, 0.3)                       # host operands
    assert np.array_equal(out, want)
    dt, dk, do = be.tensor(table), be.tensor(tok, I32), be.tensor(np.full(rows * dim + 8, GUARD, F32))
    be.embeddingForward(dt, dk, do, rows, vocab, dim, 0.3)                            # device operands
    got = do.numpy()
    assert np.array_equal(got[:rows * dim].reshape(rows, dim), want) and np.all(got[rows * dim:] == GUARD)
    free(dt, dk, do)


def test_embedding_forward_misaligned(be):
    """Operands that start one float into a block: no 16-byte access fits."""
    rng = np.random.default_rng(3)
    rows, vocab, dim = 37, 50, 64
    table, tok = rng.standard_normal(vocab * dim + 1).astype(F32), zipf_tokens(rng, rows, vocab)
    dt, dk, do = be.tensor(table), be.tensor(np.append(I32(0), tok), I32), be.tensor(np.full(rows * dim + 1, GUARD, F32))
    be.embeddingForward(dt.address + 4, dk.address + 4, do.address + 4, rows, vocab, dim, 2.0)
    got = do.numpy()
    assert got[0] == GUARD and np.array_equal(got[1:].reshape(rows, dim), ref.embedding_forward(table[1:].reshape(vocab, dim), tok, 2.0))
    free(dt, dk, do)


BACKWARD = [(1, 1, 1, "zipf"), (1, 9, 4, "zipf"), (5, 3, 7, "zipf"), (33, 100, 64, "zipf"), (777, 5000, 103, "zipf"),
            (1000, 50, 260, "zipf"), (4099, 3001, 96, "zipf"), (2500, 40, 33, "one"), (6000, 300, 20, "one"), (3000, 2, 130, "zipf"),
            (20000, 70000, 8, "flat"), (4096, 4096, 16, "each"), (64, 1000, 1030, "none"), (70001, 129, 5, "zipf"), (40000, 100000, 12, "zipf")]


def backward_tokens(rng, rows, vocab, kind):
    if kind == "one":
        return np.full(rows, vocab - 1, I32)
    if kind == "none":
        return np.full(rows, -1, I32)
    if kind == "each":
        return rng.permutation(vocab)[:rows].astype(I32)
    if kind == "flat":
        return rng.integers(0, vocab, rows).astype(I32)
    return zipf_tokens(rng, rows, vocab)


@pytest.mark.parametrize("rows,vocab,dim,kind", BACKWARD)
def test_embedding_backward(be, rows, vocab, dim, kind):
    rng = np.random.default_rng(rows + 7 * dim)
    tok = backward_tokens(rng, rows, vocab, kind)
    g = rng.standard_normal((rows, dim)).astype(F32)
    old = rng.standard_normal((vocab, dim)).astype(F32)
    dg, dk, dt = be.tensor(g), be.tensor(tok, I32), be.tensor(old)
    be.embeddingBackward(dg, dk, dt, rows, vocab, dim, 0.7, accumulate=True)
    got = dt.numpy((vocab, dim))
    want, err = ref.embedding_backward(g, tok, vocab, 0.7, old)
    ref.check(got, want, err, "accumulated")
    unused = np.ones(vocab, bool)
    unused[tok[tok >= 0]] = False
    assert np.array_equal(got[unused], old[unused])
    be.embeddingBackward(dg, dk, dt, rows, vocab, dim, 0.7)                # now the whole table, over what stood there
    first = dt.numpy((vocab, dim))
    ref.check(first, *ref.embedding_backward(g, tok, vocab, 0.7), "written")
    assert not first[unused].any()
    be.embeddingBackward(dg, dk, dt, rows, vocab, dim, 0.7)
    assert np.array_equal(dt.numpy((vocab, dim)), first)                   # the same bits again
    host = old.copy()
    be.embeddingBackward(g, tok, host, rows, vocab, dim, 0.7)
    assert np.array_equal(host, first)
    free(dg, dk, dt)


def test_embedding_backward_misaligned_and_neighbours(be):
    rng = np.random.default_rng(5)
    rows, vocab, dim = 300, 40, 64
    tok, g = zipf_tokens(rng, rows, vocab), rng.standard_normal((rows, dim)).astype(F32)
    dg = be.tensor(np.concatenate([[GUARD], g.ravel()]))
    dk, dt = be.tensor(np.append(I32(5), tok), I32), be.tensor(np.full(vocab * dim + 9, GUARD, F32))
    be.embeddingBackward(dg.address + 4, dk.address + 4, dt.address + 4, rows, vocab, dim, 1.0)
    got = dt.numpy()
    assert got[0] == GUARD and np.all(got[1 + vocab * dim:] == GUARD)
    ref.check(got[1:1 + vocab * dim].reshape(vocab, dim), *ref.embedding_backward(g, tok, vocab, 1.0))
    free(dg, dk, dt)


def test_embedding_without_rows(be):
    t = be.tensor(np.ones(12, F32))
    be.embeddingForward(t, np.zeros(0, I32), np.zeros(0, F32), 0, 3, 4)
    be.embeddingBackward(None, None, t, 0, 3, 4, accumulate=True)
    assert np.all(t.numpy() == 1)
    be.embeddingBackward(None, None, t, 0, 3, 4)
    assert not t.numpy().any()
    t.free()


def test_embedding_table_past_2_31_values(be):
    rng = np.random.default_rng(6)
    vocab, dim, rows = 270_001, 8192, 40
    table = be.tensor(vocab * dim)                                         # 8.8 GB of zeros
    last = rng.standard_normal(dim).astype(F32)
    zn.backend.check(zn.lib.zn_tensor_upload(be.handle, table.address + 4 * (vocab - 1) * dim, last.ctypes.data, dim))
    tok = np.where(np.arange(rows) % 3 == 0, vocab - 1, vocab // 2).astype(I32)
    out = np.empty((rows, dim), F32)
    be.embeddingForward(table, tok, out, rows, vocab, dim, 0.5)
    assert np.array_equal(out[tok == vocab - 1], np.tile(F32(0.5) * last, ((tok == vocab - 1).sum(), 1))) and not out[tok != vocab - 1].any()
    g = rng.standard_normal((rows, dim)).astype(F32)
    dg, dk = be.tensor(g), be.tensor(tok, I32)
    be.embeddingBackward(dg, dk, table, rows, vocab, dim, 1.0, accumulate=True)
    got = np.empty(dim, F32)
    zn.backend.check(zn.lib.zn_tensor_download(be.handle, got.ctypes.data, table.address + 4 * (vocab - 1) * dim, dim))
    sub, err = ref.embedding_backward(g, np.where(tok == vocab - 1, 0, 1).astype(I32), 2, 1.0, np.stack([last, np.zeros(dim)]))
    ref.check(got, sub[0], err[0])
    free(table, dg, dk)


# ---- token scores ------------------------------------------------------------------------------------

def run_scores(be, buf, tok, vocab, t, k, device=True):
    rows, ld = buf.shape
    out = dict(logprob=np.full(rows + 1, GUARD, F32), entropy=np.full(rows + 1, GUARD, F32), row_stats=np.full(2 * rows + 2, GUARD, F32))
    tops = (np.full(rows * k + 1, -5, I32), np.full(rows * k + 1, GUARD, F32)) if k else (None, None)
    if not device:
        be.tokenLogProbs(buf, tok, rows, vocab, **out, top_k=k, top_tokens=tops[0], top_logprobs=tops[1], temperature=t, ld=ld)
    else:
        dx, dk = be.tensor(buf), be.tensor(tok, I32)
        d = {n: be.tensor(v) for n, v in out.items()}
        dtop = (be.tensor(tops[0], I32), be.tensor(tops[1])) if k else (None, None)
        be.tokenLogProbs(dx, dk, rows, vocab, **d, top_k=k, top_tokens=dtop[0], top_logprobs=dtop[1], temperature=t, ld=ld)
        out = {n: v.numpy() for n, v in d.items()}
        if k:
            tops = dtop[0].numpy(), dtop[1].numpy()
            free(*dtop)
        free(dx, dk, *d.values())
    for v in list(out.values()) + ([tops[1]] if k else []):
        assert v[-1] == GUARD
    assert not k or tops[0][-1] == -5
    return (out["logprob"][:rows], out["entropy"][:rows], out["row_stats"][:2 * rows].reshape(rows, 2),
            tops[0][:-1].reshape(rows, k) if k else None, tops[1][:-1].reshape(rows, k) if k else None)


def check_scores(got, want, k):
    for name, g, w in zip(("logprob", "entropy", "stats"), got, want):
        ref.check(g, *w, name)
    if k:
        assert np.array_equal(got[3], want[3]), np.argwhere(got[3] != want[3])[:5]
        ref.check(got[4], *want[4], "top logprobs")


SCORES = [(1, 1, 1, 1.0, 1), (1, 5, 5, 2.0, 8), (3, 17, 20, 0.7, 17), (2, 129, 129, 1.0, 128), (5, 1000, 1003, 1.3, 3), (300, 999, 999, 1.0, 10),
          (1, 131072, 131072, 0.8, 20), (7, 50001, 50001, 1.0, 128), (2, 200003, 200010, 3.0, 64), (700, 4099, 4100, 1.0, 5),
          (1500, 257, 260, 0.5, 40), (900, 3000, 3001, 1.0, 100), (600, 1025, 1027, 1.0, 64), (600, 2048, 2048, 0.9, 128), (3, 8000, 8000, 1.0, 65), (70000, 3, 3, 1.0, 2), (64, 32768, 32768, 1.0, 0), (640, 20001, 20001, 1.0, 31), (13, 8191, 8192, 1.0, 1)]


@pytest.mark.parametrize("rows,vocab,ld,t,k", SCORES)
def test_scores(be, rows, vocab, ld, t, k):
    rng = np.random.default_rng(vocab + rows)
    buf = padded(rng, rows, vocab, ld)
    tok = rng.integers(-1, vocab, rows).astype(I32)
    want = ref.token_logprobs(buf[:, :vocab], tok, t, k)
    got = run_scores(be, buf, tok, vocab, t, k)
    check_scores(got, want, k)
    again = run_scores(be, buf, tok, vocab, t, k)
    host = run_scores(be, buf, tok, vocab, t, k, device=False)
    for a, b, c in zip(got, again, host):
        assert a is None or (np.array_equal(a, b) and np.array_equal(a, c))


def awkward_rows(rng, vocab):
    """Rows that defeat a filter or a maximum kept on the way: equal values, sorted ones, a few survivors of a mask, the
    lowest finite value as a mask, signed zeros, one overwhelming value, spread far beyond what exp can hold."""
    low = np.finfo(F32).min
    rows = [np.zeros(vocab), np.arange(vocab) * 1e-3, -np.arange(vocab) * 1e-3, np.full(vocab, 7.5)]
    r = np.full(vocab, NINF)
    r[[vocab // 3, vocab - 1]] = [1.0, 2.0]
    rows.append(r)
    r = np.full(vocab, NINF)
    r[vocab // 2] = -3.0
    rows.append(r)
    r = np.full(vocab, low)
    r[vocab // 5] = 0.5
    rows += [r, np.full(vocab, low)]
    rows.append(np.where(np.arange(vocab) % 2 == 0, 0.0, -0.0))
    r = rng.standard_normal(vocab)
    r[vocab // 4] = 300.0
    rows += [r, rng.standard_normal(vocab) * 200, np.round(rng.standard_normal(vocab) * 2)]
    r = rng.standard_normal(vocab)
    r[: vocab // 2] = NINF
    rows.append(r)
    rows.append(np.sort(rng.standard_normal(vocab)))
    r = rng.standard_normal(vocab)
    r[::97] += 50 + np.arange(len(r[::97])) * 1e-2
    rows.append(r)
    return np.asarray(rows).astype(F32)


@pytest.mark.parametrize("vocab", [37, 1000, 4096, 9001, 66000])
@pytest.mark.parametrize("k", [1, 20, 128])
def test_scores_of_awkward_rows(be, vocab, k):
    rng = np.random.default_rng(vocab)
    x = awkward_rows(rng, vocab)
    tok = np.full(len(x), vocab - 1, I32)
    check_scores(run_scores(be, x, tok, vocab, 1.0, k), ref.token_logprobs(x, tok, 1.0, k), k)
    many = np.tile(x, (60, 1))                     # enough rows that each gets one block
    mtok = np.tile(tok, 60)
    check_scores(run_scores(be, many, mtok, vocab, 1.0, k), ref.token_logprobs(many, mtok, 1.0, k), k)


@pytest.mark.parametrize("vocab", [5, 700, 30011])
def test_scores_of_rows_without_a_distribution(be, vocab):
    rng = np.random.default_rng(8)
    x = rng.standard_normal((6, vocab)).astype(F32)
    x[0] = NINF                                    # nothing left by the mask
    x[1] = NINF
    x[2, vocab // 2] = np.nan
    x[3, vocab - 1] = np.inf
    x[4] = NINF
    x[4, 0] = np.nan
    tok = np.array([vocab - 1, -1, 0, -1, 1, 2], I32)
    lp, h, st, top, tl = run_scores(be, x, tok, vocab, 1.0, 4)
    assert lp[0] == NINF and lp[1] == 0 and np.isnan(lp[2:5]).all() and np.isfinite(lp[5])
    assert h[0] == 0 and h[1] == 0 and np.isnan(h[2:5]).all()
    assert np.all(st[:2] == NINF) and np.isnan(st[2:5]).all()
    assert np.all(top[:5] == -1) and np.all(tl[:2] == NINF) and np.isnan(tl[2:5]).all()
    want = ref.token_logprobs(x[5:], tok[5:], 1.0, 4)
    check_scores([v[5:] for v in (lp, h, st, top, tl)], want, 4)


def test_scores_one_output_at_a_time(be):
    """Every output by itself gives the bits that all together give."""
    rng = np.random.default_rng(9)
    rows, vocab, k = 5, 5003, 9
    x, tok = padded(rng, rows, vocab, vocab), rng.integers(0, vocab, rows).astype(I32)
    lp, h, st, top, tl = run_scores(be, x, tok, vocab, 0.9, k)
    a = np.empty(rows, F32)
    be.tokenLogProbs(x, tok, rows, vocab, logprob=a, temperature=0.9)
    assert np.array_equal(a, lp)
    be.tokenLogProbs(x, None, rows, vocab, entropy=a, temperature=0.9)
    assert np.array_equal(a, h)
    b = np.empty((rows, 2), F32)
    be.tokenLogProbs(x, None, rows, vocab, row_stats=b, temperature=0.9)
    assert np.array_equal(b, st)
    c, d = np.empty((rows, k), I32), np.empty((rows, k), F32)
    be.tokenLogProbs(x, None, rows, vocab, top_k=k, top_tokens=c, top_logprobs=d, temperature=0.9)
    assert np.array_equal(c, top) and np.array_equal(d, tl)


def test_scores_misaligned(be):
    rng = np.random.default_rng(10)
    for shift in (1, 2, 3):
        for rows, vocab, ld in [(3, 9001, 9005), (900, 130, 131)]:
            x = padded(rng, rows, vocab, ld)
            tok = rng.integers(0, vocab, rows).astype(I32)
            dx = be.tensor(np.concatenate([np.full(shift, GUARD, F32), x.ravel()]))
            lp, c, d = np.empty(rows, F32), np.empty((rows, 7), I32), np.empty((rows, 7), F32)
            be.tokenLogProbs(dx.address + 4 * shift, tok, rows, vocab, logprob=lp, top_k=7, top_tokens=c, top_logprobs=d, ld=ld)
            want = ref.token_logprobs(x[:, :vocab], tok, 1.0, 7)
            ref.check(lp, *want[0])
            assert np.array_equal(c, want[3])
            dx.free()


GRADS = [(1, 1, 1, 1, 1.0), (1, 5, 5, 7, 2.0), (3, 17, 20, 20, 0.7), (5, 1000, 1003, 1000, 1.3), (300, 999, 999, 999, 1.0),
         (1, 131072, 131072, 131072, 0.8), (7, 50001, 50001, 50003, 1.0), (700, 4099, 4100, 4100, 1.0), (1500, 257, 260, 263, 0.5), (70000, 3, 3, 4, 1.0)]


@pytest.mark.parametrize("which", ["both", "logprob", "entropy"])
@pytest.mark.parametrize("rows,vocab,ld,ld_grad,t", GRADS)
def test_scores_backward(be, rows, vocab, ld, ld_grad, t, which):
    rng = np.random.default_rng(vocab + rows)
    buf = padded(rng, rows, vocab, ld)
    if vocab > 4:
        buf[:, 2] = NINF
    tok = rng.integers(-1, vocab, rows).astype(I32)
    gl = rng.standard_normal(rows).astype(F32) if which != "entropy" else None
    gh = rng.standard_normal(rows).astype(F32) if which != "logprob" else None
    want, err = ref.token_logprobs_backward(buf[:, :vocab], tok, t, gl, gh)
    h, st = np.empty(rows, F32), np.empty((rows, 2), F32)
    dx = be.tensor(buf)
    be.tokenLogProbs(dx, None, rows, vocab, entropy=h, row_stats=st, temperature=t, ld=ld)
    dg = be.tensor(np.full(rows * ld_grad, GUARD, F32))
    args = (tok if gl is not None else None, st, h if gh is not None else None, gl, gh)
    be.tokenLogProbsBackward(dx, *args, dg, rows, vocab, t, ld, ld_grad)
    got = dg.numpy((rows, ld_grad))
    ref.check(got[:, :vocab], want, err, which)
    assert np.all(got[:, vocab:] == GUARD)
    be.tokenLogProbsBackward(dx, *args, dx, rows, vocab, t, ld, ld)          # in place
    inp = dx.numpy((rows, ld))
    assert np.array_equal(inp[:, :vocab], got[:, :vocab]) and np.all(inp[:, vocab:] == GUARD)
    host = np.full((rows, ld_grad), GUARD, F32)
    be.tokenLogProbsBackward(buf, *args, host, rows, vocab, t, ld, ld_grad)
    assert np.array_equal(host, got)
    free(dx, dg)


def test_scores_backward_against_differences(be):
    """Central differences of the forward call.  Step h: the truncation is h^2/6 of a third derivative of order 1, the
    forward values carry about 1e-6, which the quotient turns into 1e-6 / h: with h = 0.02 both stay below 2e-4."""
    rng = np.random.default_rng(11)
    rows, vocab, t, h = 24, 24, 1.2, 0.02
    x = rng.standard_normal(vocab).astype(F32)
    st, ent = np.empty((1, 2), F32), np.empty(1, F32)
    be.tokenLogProbs(x, None, 1, vocab, entropy=ent, row_stats=st, temperature=t)
    g = np.empty((1, vocab), F32)
    be.tokenLogProbsBackward(x, np.array([5], I32), st, ent, np.array([0.7], F32), np.array([0.4], F32), g, 1, vocab, t)
    values = []
    for sign in (1, -1):
        v = np.tile(x, (rows, 1)) + sign * F32(h) * np.eye(vocab, dtype=F32)
        lp, e = np.empty(rows, F32), np.empty(rows, F32)
        be.tokenLogProbs(np.ascontiguousarray(v), np.full(rows, 5, I32), rows, vocab, logprob=lp, entropy=e, temperature=t)
        values.append(0.7 * lp.astype(np.float64) + 0.4 * e)
    assert np.max(np.abs((values[0] - values[1]) / (2 * h) - g[0])) < 2e-4


@pytest.mark.parametrize("vocab", [6, 7001])
def test_scores_backward_of_odd_rows(be, vocab):
    rng = np.random.default_rng(12)
    x = rng.standard_normal((6, vocab)).astype(F32)
    x[0] = NINF
    x[1, 3] = np.nan
    x[2, 3] = np.nan                               # but nothing asks for its gradient
    x[3, 1] = np.inf
    tok = np.array([1, 1, 1, 1, 1, -1], I32)
    gl, gh = np.array([1, 1, 0, 1, 0, 1], F32), np.array([1, 0, 0, 1, 0, 0], F32)
    h, st, g = np.empty(6, F32), np.empty((6, 2), F32), np.full((6, vocab), GUARD, F32)
    be.tokenLogProbs(x, None, 6, vocab, entropy=h, row_stats=st)
    be.tokenLogProbsBackward(x, tok, st, h, gl, gh, g, 6, vocab)
    assert not g[[0, 2, 4, 5]].any() and np.isnan(g[[1, 3]]).all()


# ---- distillation ----------------------------------------------------------------------------------------

def teacher(rng, rows, vocab, k, missing=0.2):
    ids = np.stack([rng.permutation(vocab)[:k] if vocab >= k else rng.integers(0, vocab, k) for _ in range(rows)]).astype(I32)
    ids[rng.random((rows, k)) < missing] = -1
    return ids, (rng.standard_normal((rows, k)) * 2 + 5).astype(F32)


def run_distill(be, buf, ids, u, vocab, t, w, ld_grad, in_place=False):
    rows, ld = buf.shape
    dx, di, du, dw = be.tensor(buf), be.tensor(ids, I32), be.tensor(u), be.tensor(w)
    dl = be.tensor(np.full(rows + 1, GUARD, F32))
    dg = dx if in_place else be.tensor(np.full(rows * ld_grad + 1, GUARD, F32))
    be.distillLoss(dx, di, du, rows, vocab, ids.shape[1], t, dw, dl, dg, ld, ld if in_place else ld_grad)
    loss, g = dl.numpy(), dg.numpy()
    assert loss[-1] == GUARD
    if not in_place:
        assert g[-1] == GUARD
        g = g[:-1]
        dg.free()
    g = g.reshape(rows, -1)
    assert np.all(g[:, vocab:] == GUARD)
    free(dx, di, du, dw, dl)
    return loss[:-1], g[:, :vocab]


DISTILL = [(1, 1, 1, 1, 1, 1.0), (1, 5, 5, 7, 3, 2.0), (3, 17, 20, 20, 17, 0.7), (5, 1000, 1003, 1001, 512, 1.3), (300, 999, 999, 999, 10, 1.0),
           (1, 131072, 131072, 131072, 64, 2.0), (7, 50001, 50001, 50003, 20, 1.0), (2, 200003, 200010, 200003, 100, 3.0),
           (700, 4099, 4100, 4101, 5, 1.0), (1500, 257, 260, 260, 40, 0.5), (40, 32768, 32768, 32768, 16, 4.0), (2, 460001, 460001, 460001, 9, 1.0), (70000, 3, 3, 3, 2, 1.0), (600, 20000, 20000, 20000, 300, 1.0), (200, 150001, 150001, 150001, 7, 1.0)]


@pytest.mark.parametrize("rows,vocab,ld,ld_grad,k,t", DISTILL)
def test_distill(be, rows, vocab, ld, ld_grad, k, t):
    rng = np.random.default_rng(vocab + rows)
    buf = padded(rng, rows, vocab, ld)
    ids, u = teacher(rng, rows, vocab, k)
    w = rng.standard_normal(rows).astype(F32)
    if rows > 2:
        w[1] = 0
        ids[2] = -1
    (loss, loss_err), (grad, err) = ref.distill_loss(buf[:, :vocab], ids, u, t, w)
    gl, gg = run_distill(be, buf, ids, u, vocab, t, w, ld_grad)
    ref.check(gl, loss, loss_err, "loss")
    ref.check(gg, grad, err, "gradient")
    il, ig = run_distill(be, buf, ids, u, vocab, t, w, ld_grad, in_place=True)
    assert np.array_equal(il, gl) and np.array_equal(ig, gg)
    hl, hg = np.empty(rows, F32), np.full((rows, ld_grad), GUARD, F32)
    be.distillLoss(buf, ids, u, rows, vocab, k, t, w, hl, hg, ld, ld_grad)            # host operands
    assert np.array_equal(hl, gl) and np.array_equal(hg[:, :vocab], gg) and np.all(hg[:, vocab:] == GUARD)
    be.distillLoss(buf, ids, u, rows, vocab, k, t, w, row_loss=hl, ld=ld)             # one output at a time
    assert np.array_equal(hl, gl)
    be.distillLoss(buf, ids, u, rows, vocab, k, t, w, grad_logits=hg, ld=ld, ld_grad=ld_grad)
    assert np.array_equal(hg[:, :vocab], gg)


def test_distill_duplicates_masks_and_default_weights(be):
    rng = np.random.default_rng(14)
    rows, vocab, k = 6, 3000, 8
    x = padded(rng, rows, vocab, vocab)
    x[:, 1000:1100] = NINF
    ids, u = teacher(rng, rows, 1000, k, 0)
    ids[0] = 7                                     # one token, eight times
    ids[1, ::2] = ids[1, 1::2]
    u[2, :5] = NINF                                # entries that are none
    u[3] = NINF
    u[4] = np.finfo(F32).min                       # a teacher masked by the lowest value, evenly
    (loss, le), (grad, ge) = ref.distill_loss(x, ids, u, 1.0, np.ones(rows))
    gl, gg = np.empty(rows, F32), np.empty((rows, vocab), F32)
    be.distillLoss(x, ids, u, rows, vocab, k, row_loss=gl, grad_logits=gg)
    ref.check(gl, loss, le)
    ref.check(gg, grad, ge)
    assert gl[3] == 0 and not gg[3].any()


@pytest.mark.parametrize("vocab", [40, 20011])
def test_distill_of_odd_rows(be, vocab):
    rng = np.random.default_rng(15)
    rows, k = 9, 3
    x = padded(rng, rows, vocab, vocab)
    ids, u = teacher(rng, rows, vocab, k, 0)
    w = np.full(rows, 0.5, F32)
    x[0, 5] = np.nan
    x[1, 5] = np.nan
    w[1] = 0                                       # padding may hold anything
    x[2] = NINF                                    # nothing left by the mask
    x[3, ids[3, 1]] = NINF                         # a listed token the student cannot give
    x[4, 2] = np.inf
    u[5, 1] = np.nan
    u[6, 1] = np.inf
    ids[7] = -1
    x[7, 0] = np.nan
    loss, g = run_distill(be, x, ids, u, vocab, 2.0, w, vocab)
    assert np.isnan(loss[[0, 4, 5, 6]]).all() and np.isnan(g[[0, 4, 5, 6]]).all()
    assert loss[1] == 0 and not g[1].any() and loss[7] == 0 and not g[7].any()
    assert loss[2] == np.inf and loss[3] == np.inf
    q = np.exp(u[2] / 2.0 - (u[2] / 2.0).max())
    q /= q.sum()
    want = np.zeros(vocab)
    want[ids[2]] = -q * 2.0 * 0.5
    assert np.allclose(g[2], want, rtol=64 * ref.U, atol=0)
    (_, _), (grad, err) = ref.distill_loss(x[[3, 8]], ids[[3, 8]], u[[3, 8]], 2.0, w[[3, 8]])
    ref.check(g[[3, 8]], grad, err)


@pytest.mark.parametrize("vocab", [130, 9003, 40001, 160003])
def test_distill_rows_of_all_kinds_in_one_call(be, vocab):
    """What a row is does not show in the next one of the same block: many rows, every fifth with something odd."""
    rng = np.random.default_rng(27)
    rows, k = 400, 5
    x = padded(rng, rows, vocab, vocab)
    ids, u = teacher(rng, rows, vocab, k)
    ids[:, 0] = 7
    w = np.ones(rows, F32)
    kind = np.where(np.arange(rows) % 5 == 2, rng.integers(1, 6, rows), 0)
    for r in np.nonzero(kind)[0]:
        if kind[r] == 1:
            x[r, vocab // 2] = np.nan
        elif kind[r] == 2:
            w[r] = 0
            x[r, 1] = np.inf
        elif kind[r] == 3:
            ids[r] = -1
        elif kind[r] == 4:
            x[r] = NINF
        else:
            u[r, 0] = np.nan
    loss, g = run_distill(be, x, ids, u, vocab, 1.0, w, vocab)
    again, g2 = run_distill(be, x, ids, u, vocab, 1.0, w, vocab, in_place=True)
    assert np.array_equal(loss, again, equal_nan=True) and np.array_equal(g, g2, equal_nan=True)
    fine = kind == 0
    (l, le), (grad, ge) = ref.distill_loss(x[fine], ids[fine], u[fine], 1.0, w[fine])
    ref.check(loss[fine], l, le)
    ref.check(g[fine], grad, ge)
    assert np.isnan(loss[(kind == 1) | (kind == 5)]).all() and np.isnan(g[(kind == 1) | (kind == 5)]).all()
    assert not loss[(kind == 2) | (kind == 3)].any() and not g[(kind == 2) | (kind == 3)].any()
    assert np.all(loss[kind == 4] == np.inf) and np.isfinite(g[kind == 4]).all()


def test_distill_against_differences(be):
    """As for the scores: step 0.02, truncation and the rounding of the losses both below 2e-4."""
    rng = np.random.default_rng(16)
    vocab, t, h = 20, 1.5, 0.02
    x = rng.standard_normal(vocab).astype(F32)
    ids, u = np.array([[3, 9, 9, -1]], I32), rng.standard_normal((1, 4)).astype(F32)
    g = np.empty((1, vocab), F32)
    be.distillLoss(x, ids, u, 1, vocab, 4, t, grad_logits=g)
    values = []
    for sign in (1, -1):
        v = np.ascontiguousarray(np.tile(x, (vocab, 1)) + sign * F32(h) * np.eye(vocab, dtype=F32))
        loss = np.empty(vocab, F32)
        be.distillLoss(v, np.tile(ids, (vocab, 1)), np.tile(u, (vocab, 1)), vocab, vocab, 4, t, row_loss=loss)
        values.append(loss.astype(np.float64))
    assert np.max(np.abs((values[0] - values[1]) / (2 * h) - g[0])) < 2e-4


def test_logits_past_2_31_values(be):
    """Two rows with content at the ends of a block of 2.2 thousand million logits."""
    rng = np.random.default_rng(17)
    rows, vocab = 17001, 131072
    x = be.tensor(rows * vocab)
    first, last = rng.standard_normal(vocab).astype(F32), rng.standard_normal(vocab).astype(F32)
    end = x.address + 4 * (rows - 1) * vocab
    up = lambda at, v: zn.backend.check(zn.lib.zn_tensor_upload(be.handle, at, v.ctypes.data, v.size))  # noqa: E731
    up(x.address, first)
    up(end, last)
    tok = np.zeros(rows, I32)
    tok[-1] = vocab - 1
    lp, h, st, c, d = np.empty(rows, F32), np.empty(rows, F32), np.empty((rows, 2), F32), np.empty((rows, 3), I32), np.empty((rows, 3), F32)
    be.tokenLogProbs(x, tok, rows, vocab, lp, h, st, 3, c, d)
    two = np.stack([first, last])
    want = ref.token_logprobs(two, tok[[0, -1]], 1.0, 3)
    check_scores([v[[0, -1]] for v in (lp, h, st, c, d)], want, 3)
    assert np.all(c[1:-1] == [0, 1, 2])
    gl = np.zeros(rows, F32)
    gl[[0, -1]] = 1
    be.tokenLogProbsBackward(x, tok, st, h, gl, gl, x, rows, vocab)           # in place
    got = np.empty((2, vocab), F32)
    down = lambda at, v: zn.backend.check(zn.lib.zn_tensor_download(be.handle, v.ctypes.data, at, v.size))  # noqa: E731
    down(x.address, got[0])
    down(end, got[1])
    ref.check(got, *ref.token_logprobs_backward(two, tok[[0, -1]], 1.0, [1, 1], [1, 1]))
    up(x.address, first)
    up(end, last)
    ids, u = teacher(rng, rows, 50, 4)
    w = np.zeros(rows, F32)
    w[[0, -1]] = 1
    loss = np.empty(rows, F32)
    be.distillLoss(x, ids, u, rows, vocab, 4, 1.0, w, loss, x)
    down(x.address, got[0])
    down(end, got[1])
    (l, le), (g, ge) = ref.distill_loss(two, ids[[0, -1]], u[[0, -1]], 1.0, np.ones(2))
    ref.check(loss[[0, -1]], l, le)
    ref.check(got, g, ge)
    x.free()


# ---- 4-bit weights ---------------------------------------------------------------------------------------

QUANT = [(1, 1, 32), (3, 5, 32), (8, 128, 64), (17, 129, 128), (100, 1000, 32), (257, 640, 64), (64, 4096, 128), (1003, 300, 128)]


@pytest.mark.parametrize("n,k,group", QUANT)
def test_quantize4(be, n, k, group):
    rng = np.random.default_rng(n + k)
    w = rng.standard_normal((k, n)).astype(F32)
    w[:, 0] = 0
    if n > 2:
        w[k // 2, 1] = np.nan
        w[k - 1, 2] = np.inf
    codes, scales = ref.quantize4(w, group)
    (ps, ss) = zn.Backend.packed4_shape(n, k, group)
    p, s = np.zeros(ps, U32), np.zeros(ss, F32)
    be.quantize4(w, p, s, n, k, group)
    assert np.array_equal(s, scales, equal_nan=True)
    assert np.array_equal(p, ref.pack4(codes))


MATMUL4 = [(1, 1, 1, 32), (1, 7, 5, 64), (1, 64, 128, 128), (1, 4096, 4096, 64), (2, 100, 257, 32), (3, 1003, 640, 64), (8, 333, 1000, 128),
           (5, 17, 4000, 32), (16, 129, 513, 64), (17, 64, 300, 32), (2, 12000, 2000, 64), (9, 10001, 1100, 32), (6, 19300, 4100, 128), (40, 200, 1025, 128), (1, 20001, 512, 128), (7, 50, 8192, 128), (1, 31, 30000, 64)]


@pytest.mark.parametrize("act", ["linear", "relu", "gelu"])
@pytest.mark.parametrize("rows,n,k,group", MATMUL4)
def test_matmul4(be, rows, n, k, group, act):
    rng = np.random.default_rng(n + k)
    codes = rng.integers(0, 16, (n, -(-k // 128) * 128))                     # what stands past k is ignored
    scales = (rng.random((n, -(-k // group))) * 0.1 + 0.01).astype(F32)
    x = (rng.standard_normal((rows, k)) * np.exp(rng.standard_normal((rows, 1)) * 3)).astype(F32)
    bias = rng.standard_normal(n).astype(F32) if act != "linear" else None
    y, err = ref.matmul4(x, codes, scales, k, group, bias)
    if act == "relu":
        y = np.maximum(y, 0)
    elif act == "gelu":                            # slope at most 1.13; its own roundings stay below 16 U of the input
        err = 1.2 * err + 16 * ref.U * np.abs(y) + 16 * ref.U
        y = 0.5 * y * (1 + np.tanh(np.float64(F32(0.7978845608)) * (y + np.float64(F32(0.044715)) * y ** 3)))
    dx, dp, ds = be.tensor(x), be.tensor(ref.pack4(codes), U32), be.tensor(scales)
    db, dy = (be.tensor(bias) if bias is not None else None), be.tensor(np.full(rows * n + 1, GUARD, F32))
    be.matMul4BiasAct(dx, dp, ds, db, dy, rows, n, k, group, zn.Activation[act])
    got = dy.numpy()
    assert got[-1] == GUARD
    ref.check(got[:-1].reshape(rows, n), y, err + 2 * ref.U * np.abs(y), f"{rows}x{n}x{k}")
    be.matMul4BiasAct(dx, dp, ds, db, dy, rows, n, k, group, zn.Activation[act])
    assert np.array_equal(dy.numpy(), got)
    host = np.empty((rows, n), F32)
    be.matMul4BiasAct(x, ref.pack4(codes), scales, bias, host, rows, n, k, group, zn.Activation[act])
    assert np.array_equal(host.ravel(), got[:-1])
    free(dx, dp, ds, dy)
    if db:
        db.free()


def test_matmul4_all_activations(be):
    rng = np.random.default_rng(20)
    rows, n, k, group = 3, 40, 96, 32
    w = rng.standard_normal((k, n)).astype(F32) * 0.2
    (ps, ss) = zn.Backend.packed4_shape(n, k, group)
    p, s = np.zeros(ps, U32), np.zeros(ss, F32)
    be.quantize4(w, p, s, n, k, group)
    codes, _ = ref.quantize4(w, group)
    x, bias = rng.standard_normal((rows, k)).astype(F32), rng.standard_normal(n).astype(F32)
    deq = np.ascontiguousarray(ref.dequantize4(codes, s, k, group), F32)
    for act in zn.Activation:
        y, want = np.empty((rows, n), F32), np.empty((rows, n), F32)
        be.matMul4BiasAct(x, p, s, bias, y, rows, n, k, group, act)
        be.matMulBiasAct(x, deq, bias, want, rows, n, k, act)          # the dense call on the weights the codes stand for
        # both sides: k + 64 roundings of sums of size about 10 at most, through a slope of at most 1.13
        assert np.max(np.abs(y - want)) <= 2 * 1.13 * (k + 64) * 2 * ref.U * 10, act.name


def test_matmul4_exact_in_x(be):
    """All 24 bits of x count: one weight of code 9 and scale 1 returns x itself, subnormals of the parts aside."""
    rng = np.random.default_rng(21)
    k = n = 64
    codes = np.full((n, 128), 8)
    codes[np.arange(n), np.arange(n)] = 9
    x = (rng.standard_normal((4, k)) * np.exp(rng.uniform(-30, 30, (4, k)))).astype(F32)
    x[0, :3] = [np.finfo(F32).max, -np.finfo(F32).max, 1.0]
    y = np.empty((4, n), F32)
    be.matMul4BiasAct(x, ref.pack4(codes), np.ones((n, 2), F32), None, y, 4, n, k, 32, zn.Activation.linear)
    assert np.array_equal(y, x)


def test_matmul4_of_inf_and_nan(be):
    """As the formula has it: infinity times a zero code is NaN, times another code infinity; other rows do not notice."""
    n, k = 20, 70
    codes = np.full((n, 128), 11)
    codes[3] = 8
    codes[4] = 5
    x = np.ones((4, k), F32)
    x[1, 69] = np.inf
    x[2, 0] = np.nan
    y = np.empty((4, n), F32)
    be.matMul4BiasAct(x, ref.pack4(codes), np.ones((n, 3), F32), None, y, 4, n, k, 32, zn.Activation.linear)
    want = np.full(n, 3.0 * k)
    want[3], want[4] = 0, -3.0 * k
    assert np.array_equal(y[0], want) and np.array_equal(y[3], want)
    assert np.isnan(y[2]).all() and np.isnan(y[1, 3]) and y[1, 4] == -np.inf and np.all(np.delete(y[1], [3, 4]) == np.inf)


# ---- refusals, bad ids, contexts, the whole run ----------------------------------------------------------

def refused(status, f, *args, **kw):
    with pytest.raises(zn.ZnError) as ei:
        f(*args, **kw)
    assert ei.value.status == status, ei.value


def test_refusals(be):
    INVALID, SHAPE = 1, 7
    f = np.zeros(64, F32)
    i = np.zeros(64, I32)
    u = np.zeros(64, U32)
    o = np.zeros(64, F32)
    refused(INVALID, be.embeddingForward, None, i, o, 2, 4, 8)
    refused(INVALID, be.embeddingForward, f, None, o, 2, 4, 8)
    refused(INVALID, be.embeddingForward, f, i, f, 2, 4, 8)                          # output over the table
    refused(SHAPE, be.embeddingForward, f, i, o, 2, 0, 8)
    refused(SHAPE, be.embeddingBackward, f, i, o, 2, 4, 0)
    refused(INVALID, be.embeddingBackward, f, i, None, 2, 4, 8)
    refused(INVALID, be.embeddingBackward, f, i, f, 2, 4, 8)
    refused(INVALID, be.tokenLogProbs, f, i, 2, 8)                                   # tokens without logprob
    refused(INVALID, be.tokenLogProbs, f, None, 2, 8)                                # nothing asked for
    refused(INVALID, be.tokenLogProbs, f, None, 2, 8, logprob=o)
    refused(INVALID, be.tokenLogProbs, f, None, 2, 8, top_k=2, top_tokens=i)
    refused(INVALID, be.tokenLogProbs, f, None, 2, 8, entropy=o, top_tokens=i, top_logprobs=o[8:])
    refused(INVALID, be.tokenLogProbs, f, None, 2, 8, top_k=129, top_tokens=i, top_logprobs=o)
    refused(INVALID, be.tokenLogProbs, f, None, 2, 8, entropy=f)
    refused(INVALID, be.tokenLogProbs, f, None, 2, 8, entropy=o, row_stats=o)        # two outputs on one another
    refused(SHAPE, be.tokenLogProbs, f, None, 2, 8, entropy=o, ld=7)
    refused(SHAPE, be.tokenLogProbs, f, None, 2, 0, entropy=o)
    for t in (0.0, -1.0, np.inf, np.nan, 9e-5, 1.1e4):
        refused(INVALID, be.tokenLogProbs, f, None, 2, 8, entropy=o, temperature=t)
        refused(INVALID, be.tokenLogProbsBackward, f, i, f, None, f, None, o, 2, 8, t)
        refused(INVALID, be.distillLoss, f, i, f, 2, 8, 2, t, grad_logits=o)
    refused(INVALID, be.tokenLogProbsBackward, f, i, f, None, None, None, o, 2, 8)
    refused(INVALID, be.tokenLogProbsBackward, f, None, f, None, f, None, o, 2, 8)
    refused(INVALID, be.tokenLogProbsBackward, f, i, f, None, None, f, o, 2, 8)      # entropy gradient without the entropy
    refused(INVALID, be.tokenLogProbsBackward, f, i, None, None, f, None, o, 2, 8)
    refused(INVALID, be.tokenLogProbsBackward, f, i, o[32:], None, f[40:], None, f, 2, 8, ld=8, ld_grad=9)   # in place at another pitch
    refused(INVALID, be.tokenLogProbsBackward, f, i, o, None, o[8:], None, f[1:], 2, 8)                      # shifted by one
    refused(SHAPE, be.tokenLogProbsBackward, f, i, f, None, f, None, o, 2, 8, ld_grad=7)
    refused(INVALID, be.distillLoss, f, i, f, 2, 8, 2)
    refused(INVALID, be.distillLoss, f, None, f, 2, 8, 2, row_loss=o)
    refused(INVALID, be.distillLoss, f, i, None, 2, 8, 2, row_loss=o)
    refused(SHAPE, be.distillLoss, f, i, f, 2, 8, 0, row_loss=o)
    refused(SHAPE, be.distillLoss, f, i, f, 2, 8, 513, row_loss=o)
    refused(SHAPE, be.distillLoss, f, i, f, 2, 8, 2, row_loss=o, ld=4)
    refused(INVALID, be.distillLoss, f, i, o, 2, 8, 2, row_loss=o)                   # loss over the teacher
    refused(INVALID, be.quantize4, f, u, o, 2, 8, 16)
    refused(INVALID, be.quantize4, f, None, o, 2, 8, 32)
    refused(SHAPE, be.quantize4, f, u, o, 0, 8, 32)
    refused(INVALID, be.matMul4BiasAct, f, u, o, None, o, 1, 2, 8, 32, 0)            # output over the scales
    refused(INVALID, be.matMul4BiasAct, f, u, f, None, o, 1, 2, 8, 33, 0)
    refused(SHAPE, be.matMul4BiasAct, f, u, f, None, o, 1, 0, 8, 32, 0)
    assert zn.lib.zn_matmul4_bias_act(be.handle, f.ctypes.data, u.ctypes.data, f.ctypes.data, None, o.ctypes.data, 1, 2, 8, 32, 9) == INVALID
    d = be.tensor(np.zeros(64, U32), U32)
    refused(INVALID, be.matMul4BiasAct, f, d.address + 4, f, None, o, 1, 2, 8, 32, 0)       # packed weights not on 16 bytes
    refused(INVALID, be.embeddingForward, d.address + 2, i, o, 1, 2, 8)                     # floats not on 4 bytes
    d.free()
    # rows == 0 does nothing, whatever the pointers
    be.tokenLogProbs(None, None, 0, 8, entropy=o)
    be.distillLoss(None, None, None, 0, 8, 2, row_loss=o)
    be.matMul4BiasAct(None, None, None, None, None, 0, 2, 8, 32, 0)
    assert not o.any()


def test_ids_past_the_vocabulary_are_reported_once_and_reach_nothing(be):
    rng = np.random.default_rng(22)
    vocab, dim, rows = 11, 6, 4
    bad = np.array([2, 11, 2_000_000_000, 0], I32)
    table, out = rng.standard_normal((vocab, dim)).astype(F32), np.full((rows, dim), GUARD, F32)
    refused(1, be.embeddingForward, table, bad, out, rows, vocab, dim)
    be.endCommandBatch()                                                        # reported once
    assert np.array_equal(out[[0, 3]], table[[2, 0]]) and not out[1:3].any()
    g, dt = rng.standard_normal((rows, dim)).astype(F32), be.tensor(vocab * dim)
    be.embeddingBackward(be.tensor(g), be.tensor(bad, I32), dt, rows, vocab, dim)     # device operands: enqueued
    refused(1, be.endCommandBatch)
    ref.check(dt.numpy((vocab, dim)), *ref.embedding_backward(g, np.array([2, -1, -1, 0]), vocab, 1.0))
    x, lp = rng.standard_normal((rows, vocab)).astype(F32), np.empty(rows, F32)
    refused(1, be.tokenLogProbs, x, bad, rows, vocab, logprob=lp)
    assert np.isnan(lp[1:3]).all() and np.isfinite(lp[[0, 3]]).all()
    h, st, gx = np.empty(rows, F32), np.empty((rows, 2), F32), np.empty((rows, vocab), F32)
    be.tokenLogProbs(x, None, rows, vocab, entropy=h, row_stats=st)
    one = np.ones(rows, F32)
    refused(1, be.tokenLogProbsBackward, x, bad, st, h, one, one, gx, rows, vocab)
    ref.check(gx, *ref.token_logprobs_backward(x, np.array([2, -1, -1, 0]), 1.0, one, one))
    ids = np.array([[1, 2], [3, 11], [1_000_000, -1], [4, -1]], I32)
    loss = np.empty(rows, F32)
    refused(1, be.distillLoss, x, ids, np.zeros((rows, 2), F32), rows, vocab, 2, row_loss=loss, grad_logits=gx)
    assert np.isnan(loss[1:3]).all() and np.isfinite(loss[[0, 3]]).all() and not gx[1:3].any() and gx[0].any()
    be.endCommandBatch()
    dt.free()


def test_two_contexts_at_once():
    """Two contexts work on one GPU at the same time, each in its own scratch; neither changes the other's results."""
    rng = np.random.default_rng(23)
    a, b = zn.Backend(0), zn.Backend(0)
    rows, vocab, k, dim = 6, 70001, 30, 64

    def calls(be, x, tok, tops, lp, tt, tl, g, ids, u, gx, dg, dt):
        be.tokenLogProbs(x, tok, rows, vocab, logprob=lp, top_k=k, top_tokens=tt, top_logprobs=tl)
        be.distillLoss(x, ids, u, rows, vocab, 5, grad_logits=gx)
        be.embeddingBackward(dg, tops, dt, 3000, 900, dim)

    sets = []
    for be in (a, b):
        x = rng.standard_normal((rows, vocab)).astype(F32)
        ids, u = teacher(rng, rows, vocab, 5)
        tok, tops, dg = rng.integers(0, vocab, rows), zipf_tokens(rng, 3000, 900), rng.standard_normal((3000, dim)).astype(F32)
        sets.append((be, be.tensor(x), be.tensor(tok, I32), be.tensor(tops, I32), be.tensor(rows), be.tensor(rows * k, I32), be.tensor(rows * k),
                     None, be.tensor(ids, I32), be.tensor(u), be.tensor(rows * vocab), be.tensor(dg), be.tensor(900 * dim)))
    outs = (4, 5, 6, 10, 12)
    alone = []
    for s in sets:
        calls(*s)
        alone.append([s[i].numpy() for i in outs])
    for _ in range(20):
        for s in sets:
            calls(*s)
    for s, w in zip(sets, alone):
        for i, v in zip(outs, w):
            assert np.array_equal(s[i].numpy(), v)
    a.deinit()
    b.deinit()


def test_calls_between_submitted_training_steps(be):
    """Steps in flight use the context's other streams and their scratch; calls in between give what they give alone, and
    the network trains as it does undisturbed."""
    rng = np.random.default_rng(28)
    rows, vocab, k = 3, 60001, 20
    x, tok = padded(rng, rows, vocab, vocab), rng.integers(0, vocab, rows).astype(I32)
    emb, g = zipf_tokens(rng, 5000, 300), rng.standard_normal((5000, 64)).astype(F32)
    dx, dk, de, dg = be.tensor(x), be.tensor(tok, I32), be.tensor(emb, I32), be.tensor(g)
    lp, tt, tl, dt = be.tensor(rows), be.tensor(rows * k, I32), be.tensor(rows * k), be.tensor(300 * 64)
    xin, t = rng.standard_normal((256, 96)).astype(F32), rng.standard_normal((256, 40)).astype(F32)
    w = [rng.standard_normal((96, 80)).astype(F32) * F32(0.1), rng.standard_normal((80, 40)).astype(F32) * F32(0.1)]

    def train(between):
        net = zn.Network(be, zn.Precision.FP32_SIMT)
        net.addDense(96, 80, "relu")
        net.addDense(80, 40, "linear")
        for i in range(2):
            net.setWeights(i, w[i], np.zeros(w[i].shape[1], F32))
        net.setOptimizer(zn.Adam())
        losses, flying = [], 0
        for _ in range(8):
            net.submitStep(hx, ht, 256, 1e-3, zn.Loss.mse)
            flying += 1
            if between:
                be.tokenLogProbs(dx, dk, rows, vocab, logprob=lp, top_k=k, top_tokens=tt, top_logprobs=tl)
                be.embeddingBackward(dg, de, dt, 5000, 300, 64)
            if flying == 2:
                losses.append(net.waitStep())
                flying -= 1
        losses.append(net.waitStep())
        out = [net.getWeights(i)[0] for i in range(2)]
        net.deinit()
        return losses, out

    hx, ht = be.host_alloc(xin.shape), be.host_alloc(t.shape)
    hx[:], ht[:] = xin, t
    alone, weights = train(False)
    mixed, mixed_weights = train(True)
    assert alone == mixed and all(np.array_equal(a, b) for a, b in zip(weights, mixed_weights))
    want = ref.token_logprobs(x, tok, 1.0, k)
    ref.check(lp.numpy(), *want[0])
    assert np.array_equal(tt.numpy((rows, k)), want[3])
    ref.check(dt.numpy((300, 64)), *ref.embedding_backward(g, emb, 300, 1.0))
    free(dx, dk, de, dg, lp, tt, tl, dt)


def test_small_call_after_a_large_one_in_the_same_scratch(be):
    rng = np.random.default_rng(24)
    for rows, vocab, dim in [(30000, 40000, 16), (50, 30, 16), (3000, 2000, 40)]:
        tok, g = zipf_tokens(rng, rows, vocab), rng.standard_normal((rows, dim)).astype(F32)
        got = np.empty((vocab, dim), F32)
        be.embeddingBackward(g, tok, got, rows, vocab, dim)
        ref.check(got, *ref.embedding_backward(g, tok, vocab, 1.0))
    for rows, vocab, k in [(3, 150000, 128), (1, 40, 5), (2, 30000, 2)]:
        x, tok = padded(rng, rows, vocab, vocab), rng.integers(0, vocab, rows).astype(I32)
        check_scores(run_scores(be, x, tok, vocab, 1.0, k), ref.token_logprobs(x, tok, 1.0, k), k)


def test_training_run(be):
    """Lookup, a hidden layer, logits, distillation and everything back to the table, as a program strings them
    together on device tensors; against the same in float64."""
    rng = np.random.default_rng(25)
    rows, vocab, dim, k, t = 96, 701, 48, 9, 2.0
    scale = float(np.sqrt(dim))
    table, w1 = (rng.standard_normal((vocab, dim)) * 0.1).astype(F32), (rng.standard_normal((dim, dim)) * 0.2).astype(F32)
    b1, wo = (rng.standard_normal(dim) * 0.1).astype(F32), (rng.standard_normal((dim, vocab)) * 0.2).astype(F32)
    tok = zipf_tokens(rng, rows, vocab)
    ids, u = teacher(rng, rows, vocab, k)
    w = np.where(tok >= 0, 1.0 / rows, 0.0).astype(F32)
    d = {n: be.tensor(v) for n, v in dict(table=table, w1=w1, b1=b1, wo=wo, u=u, w=w).items()}
    dtok, dids = be.tensor(tok, I32), be.tensor(ids, I32)
    e, hid, logits, loss = be.tensor(rows * dim), be.tensor(rows * dim), be.tensor(rows * vocab), be.tensor(rows)
    gh, gpre, ge, gwo, gw1, gt = (be.tensor(c) for c in (rows * dim, rows * dim, rows * dim, dim * vocab, dim * dim, vocab * dim))
    be.embeddingForward(d["table"], dtok, e, rows, vocab, dim, scale)
    be.matMulBiasAct(e, d["w1"], d["b1"], hid, rows, dim, dim, zn.Activation.tanh)
    be.matMul(hid, d["wo"], logits, rows, vocab, dim)
    be.distillLoss(logits, dids, d["u"], rows, vocab, k, t, d["w"], loss, logits)        # the gradient takes the logits' place
    be.matMulTransposeA(hid, logits, gwo, dim, vocab, rows)
    be.matMulTransposeB(logits, d["wo"], gh, rows, dim, vocab)
    be.activationBackward(zn.Activation.tanh, hid, gh, gpre)
    be.matMulTransposeA(e, gpre, gw1, dim, dim, rows)
    be.matMulTransposeB(gpre, d["w1"], ge, rows, dim, dim)
    be.embeddingBackward(ge, dtok, gt, rows, vocab, dim, scale)
    be.endCommandBatch()
    f = lambda v: v.astype(np.float64)  # noqa: E731
    e64 = np.where(tok[:, None] >= 0, scale * f(table)[np.maximum(tok, 0)], 0)
    h64 = np.tanh(e64 @ f(w1) + b1)
    (l64, _), (gl64, _) = ref.distill_loss(h64 @ f(wo), ids, u, t, w)
    gh64 = gl64 @ f(wo).T
    gp64 = gh64 * (1 - h64 ** 2)
    gt64 = ref.embedding_backward(gp64 @ f(w1).T, tok, vocab, scale)[0]
    for name, got, want in (("loss", loss, l64), ("wo", gwo, h64.T @ gl64), ("w1", gw1, e64.T @ gp64), ("table", gt, gt64)):
        g = got.numpy(want.shape)
        # six float32 stages, each a sum of up to 701 terms: 6 * 701 U = 2.5e-4 of the largest value at the very most
        assert np.max(np.abs(g - want)) <= 6 * 701 * ref.U * np.abs(want).max(), name


def test_serving_run_feeds_a_teacher(be):
    """Lookup, a 4-bit output layer and the best alternatives of each row, which then teach a dense student."""
    rng = np.random.default_rng(26)
    rows, vocab, dim, k, group = 5, 1501, 256, 12, 64
    table, wo = rng.standard_normal((vocab, dim)).astype(F32), rng.standard_normal((dim, vocab)).astype(F32) * F32(0.1)
    tok = rng.integers(0, vocab, rows).astype(I32)
    (ps, ss) = zn.Backend.packed4_shape(vocab, dim, group)
    dw, dt, dtok = be.tensor(wo), be.tensor(table), be.tensor(tok, I32)
    dp, ds, x, logits = be.tensor(ps[0] * ps[1], U32), be.tensor(ss[0] * ss[1]), be.tensor(rows * dim), be.tensor(rows * vocab)
    tt, tl, lp = be.tensor(rows * k, I32), be.tensor(rows * k), be.tensor(rows)
    be.quantize4(dw, dp, ds, vocab, dim, group)
    be.embeddingForward(dt, dtok, x, rows, vocab, dim)
    be.matMul4BiasAct(x, dp, ds, None, logits, rows, vocab, dim, group, zn.Activation.linear)
    be.tokenLogProbs(logits, dtok, rows, vocab, logprob=lp, top_k=k, top_tokens=tt, top_logprobs=tl)
    l32 = logits.numpy((rows, vocab))
    want = ref.token_logprobs(l32, tok, 1.0, k)
    assert np.array_equal(tt.numpy((rows, k)), want[3])
    ref.check(tl.numpy((rows, k)), *want[4])
    ref.check(lp.numpy(), *want[0])
    codes, scales = ref.quantize4(wo, group)
    y, err = ref.matmul4(table[tok], codes, scales, dim, group, None)
    ref.check(l32, y, err)
    student = padded(rng, rows, vocab, vocab)
    dsx, loss = be.tensor(student), be.tensor(rows)
    be.distillLoss(dsx, tt, tl, rows, vocab, k, 1.0, None, loss, dsx)
    (l, le), (g, ge) = ref.distill_loss(student, tt.numpy((rows, k)), tl.numpy((rows, k)), 1.0, np.ones(rows))
    ref.check(loss.numpy(), l, le)
    ref.check(dsx.numpy((rows, vocab)), g, ge)
