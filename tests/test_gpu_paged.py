"""GPU tests of the paged cache: append, attention of new tokens (causal, window,
sinks, grouped heads), attention weights, eviction and gather, against plain
64-bit evaluations of the formulas in include/kvforge.h.

Every cache is filled with NaN before its tokens are written, so a kernel that
reads a slot that no query sees gives a wrong result.

Tolerances (derived, not fitted). With u the output type's unit roundoff, w =
2^-24, A = sum_j p_j |v_j| for an output element and S = scale * sum_d |q_d k_d|
at its largest over the seen slots:
  scores: a sum of D products in f32, scaled: off by at most (D + 4) w S, which
    changes every p_j by that factor at most, numerator and sum: 2 (D + 4) w S A;
  exp2 and the rescaling by 2^(m - m'): 2 ulp each, one per tile: 4 w (n / 64 + 2) A;
  the sum of n terms: n w A;
  numerators rounded to the pool's type: u_p A (u_p = u for 16-bit pools, 0 for
    f32); in f16 numerators below 2^-14 of the largest lose up to 2^-25 each: the
    n of them 2^-25 n max|v| / l, with l >= 2^-8 where the running maximum may
    lag by 2^8;
  the final rounding: u |out|.
lse: (D + 4) w S + 4 w (n / 64 + 2) + n w + w |lse|. A weight: each term of its sum of r is
off by the same factors as p, and the sum by r w."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

W = 2.0 ** -24
UNIT = {torch.float32: W, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=_gen(seed), device="cuda") * scale).to(dtype)


class World:
    """A cache whose unwritten rows are NaN, its sequences (old tokens written
    through append), and the plain copies of their keys and values."""

    def __init__(self, kvf, lens, heads, dim, dtype, page=16, layers=1, seed=0, spare=3, scatter=True, big=1.0):
        self.lens, self.H, self.D, self.dtype = lens, heads, dim, dtype
        total = [a + b for a, b in lens]
        need = [-(-t // page) for t in total]
        P = sum(need) + spare
        self.cache = kvf.PagedKVCache(P, heads, dim, page_size=page, num_layers=layers, dtype=dtype)
        for t in (self.cache.keys, self.cache.values, self.cache.weights):
            t.fill_(float("nan"))
        order = np.random.RandomState(seed).permutation(P).tolist() if scatter else list(range(P))
        self.seqs, at = [], 0
        for n in need:
            self.seqs.append(self.cache.add(0, pages=order[at:at + n]))
            at += n
        self.k = [_randn((t, heads, dim), dtype, seed + 7 * i + 1, big) for i, t in enumerate(total)]
        self.v = [_randn((t, heads, dim), dtype, seed + 7 * i + 2) for i, t in enumerate(total)]
        b = self.cache.extend(self.seqs, [a for a, _ in lens])
        for layer in range(layers):
            self.cache.append(b, torch.cat([k[:a] for k, (a, _) in zip(self.k, lens)]),
                              torch.cat([v[:a] for v, (a, _) in zip(self.v, lens)]), layer)

    def step(self, query_heads, window=0, sinks=0, layer=0, seed=99):
        new = [c for _, c in self.lens]
        self.batch = self.cache.extend(self.seqs, new, query_heads, window, sinks)
        self.cache.append(self.batch, torch.cat([k[a:] for k, (a, _) in zip(self.k, self.lens)]),
                          torch.cat([v[a:] for v, (a, _) in zip(self.v, self.lens)]), layer)
        return _randn((sum(new), query_heads, self.D), self.dtype, seed)


def seen(n, c, window, sinks):
    a = torch.arange(n - c, n, device="cuda")[:, None]
    j = torch.arange(n, device="cuda")[None]
    s = j <= a
    if window:
        s &= (j > a - window) | (j < sinks)
    return s


def reference(k, v, q, scale, window, sinks, dtype):
    """One sequence in 64 bits: out [c, Hq, D], lse [c, Hq], weight sums [H, n], and
    the bounds of their errors. k, v [n, H, D], q [c, Hq, D]."""
    n, H, D = k.shape
    c, Hq, _ = q.shape
    G = Hq // H
    see = seen(n, c, window, sinks)
    out = torch.zeros((c, Hq, D), dtype=torch.float64, device="cuda")
    lse = torch.full((c, Hq), -math.inf, dtype=torch.float64, device="cuda")
    tol_out, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    wsum = torch.zeros((H, n), dtype=torch.float64, device="cuda")
    tol_w = torch.zeros_like(wsum)
    u = UNIT[dtype]
    for h in range(Hq):
        kd, vd, qd = k[:, h // G].double(), v[:, h // G].double(), q[:, h].double()
        s = (qd @ kd.T * scale).masked_fill(~see, -math.inf)
        S = torch.where(see, qd.abs() @ kd.abs().T * abs(scale), 0.0).nan_to_num(0, 0, 0).amax(1) if n else qd.sum(1) * 0
        m = s.amax(1) if n else qd.sum(1) - math.inf
        ok = m > -math.inf
        p = torch.where(ok[:, None], torch.exp(s - torch.where(ok, m, 0.0)[:, None]), 0.0)
        l = p.sum(1)
        div = torch.where(l == 0, 1.0, l)
        # what a row does not see contributes nothing, whatever it holds
        vis = p > 0
        num = torch.zeros((c, D), dtype=torch.float64, device="cuda")
        fin = torch.isfinite(vd).all(1)
        num = p[:, fin] @ vd[fin]
        for j in torch.nonzero(~fin).flatten().tolist():
            num += torch.where(vis[:, j, None], p[:, j, None] * vd[j], 0.0)
        out[:, h] = num / div[:, None]
        lse[:, h] = torch.where(ok, m + torch.log(div), -math.inf)
        p = p / div[:, None]
        A = p[:, fin] @ vd[fin].abs()
        e = (D + 4) * W * S + 4 * W * (n / 64 + 2) + n * W
        up = 0.0 if dtype == torch.float32 else u
        vmax = vd[fin].abs().max() if fin.any() else 0.0
        low = n * 2.0 ** -25 * 2.0 ** 8 * vmax / div[:, None] if dtype == torch.float16 else 0.0
        tol_out[:, h] = (2 * e[:, None] + up) * A + u * out[:, h].abs() + low
        tol_lse[:, h] = e + W * lse[:, h].abs().nan_to_num(0, 0, 0)
        wsum[h // G] += p.sum(0)
        tol_w[h // G] += (2 * e[:, None] * p).sum(0) + c * G * W * p.sum(0)
    return out, lse, wsum, tol_out, tol_lse, tol_w


def close(got, want, tol, what=""):
    got = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), what
    off = (got - want).abs()[fin] - tol[fin]
    assert off.numel() == 0 or off.max() <= 1e-30, (what, float(off.max()), float((got - want).abs()[fin].max()))


def check(w, q, window=0, sinks=0, scale=None, decay=None, layer=0, before=None):
    cache = w.cache
    got, lse = cache.attend(w.batch, q, layer, scale=scale, decay=decay, return_lse=True)
    sc = scale if scale is not None else 1.0 / math.sqrt(w.D)
    at = 0
    for i, (seq, (a, c)) in enumerate(zip(w.seqs, w.lens)):
        o, z, s, to, tz, ts = reference(w.k[i], w.v[i], q[at:at + c], sc, window, sinks, w.dtype)
        close(got[at:at + c], o, to, f"out of sequence {i}")
        close(lse[at:at + c], z, tz, f"lse of sequence {i}")
        if decay is not None and c:
            pages = torch.tensor(cache.pages(seq), device="cuda", dtype=torch.long)
            new = cache.weights[layer, pages].transpose(0, 1).reshape(w.H, -1)[:, :a + c]
            old = 0.0 if before is None else before[i].double()
            close(new, decay * old + s, ts + 4 * W * (abs(decay * old) + s), f"weights of sequence {i}")
        at += c
    return got, lse


F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# (sequences as (cached, new) tokens, KV heads, group, head_dim, page)
SHAPES = [
    ([(0, 1)], 1, 1, 64, 16),
    ([(0, 1), (1, 1), (15, 1), (16, 1), (17, 1), (63, 1), (64, 1), (127, 1), (128, 1)], 2, 4, 128, 16),
    ([(2000, 1), (0, 0), (5, 0), (700, 1)], 8, 4, 128, 64),
    ([(4095, 1)], 2, 8, 64, 128),
    ([(900, 1), (33, 1)], 1, 16, 128, 32),
    ([(500, 3), (100, 4), (0, 2)], 2, 5, 96, 32),
    ([(1000, 7)], 2, 7, 128, 16),
    ([(0, 300)], 2, 1, 128, 64),
    ([(0, 128)], 1, 1, 64, 128),
    ([(77, 129), (0, 1), (300, 256)], 2, 2, 80, 64),
    ([(1000, 257)], 2, 3, 128, 32),
    ([(640, 512)], 1, 4, 64, 16),
    ([(3, 33)], 2, 8, 32, 16),
    ([(130, 60)], 1, 40, 128, 16),
    ([(1500, 1), (10, 700), (0, 5), (300, 40)], 4, 4, 128, 64),
]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", range(len(SHAPES)))
def test_attention(kvf, dtype, case):
    lens, H, G, D, page = SHAPES[case]
    w = World(kvf, lens, H, D, dtype, page, seed=case)
    check(w, w.step(H * G), decay=0.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (64, 33), (1000, 130), (129, 500)])
@pytest.mark.parametrize("case", [1, 2, 5, 10, 11, 14])
def test_window_and_sinks(kvf, dtype, window, sinks, case):
    lens, H, G, D, page = SHAPES[case]
    w = World(kvf, lens, H, D, dtype, page, seed=case + 50)
    check(w, w.step(H * G, window, sinks), window, sinks, decay=0.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [1, 8, 20, 33, 72, 104, 112, 120, 136, 256])
def test_head_dims(kvf, dtype, D):
    w = World(kvf, [(200, 1), (50, 70), (10, 3)], 2, D, dtype, 32, seed=D)
    check(w, w.step(4), decay=0.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
def test_scales(kvf, dtype, scale):
    w = World(kvf, [(300, 1), (50, 70)], 2, 64, dtype, 32, seed=5)
    check(w, w.step(8), scale=scale, decay=0.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_large_scores(kvf, dtype):
    """Scores in the hundreds: the running maximum moves far, most terms vanish."""
    w = World(kvf, [(3000, 1), (1000, 200)], 2, 128, dtype, 32, seed=6, big=40.0)
    # growing norms, so that the maximum keeps rising along the sequence
    for i, (a, c) in enumerate(w.lens):
        w.k[i] *= torch.linspace(0.01, 1.0, a + c, device="cuda")[:, None, None].to(dtype)
    b = w.cache.batch(w.seqs, [a for a, _ in w.lens])
    w.cache.append(b, torch.cat([k[:a] for k, (a, _) in zip(w.k, w.lens)]),
                   torch.cat([v[:a] for v, (a, _) in zip(w.v, w.lens)]))
    check(w, w.step(8), decay=0.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("queries", [6, 70, 300])
def test_rows_that_see_nothing(kvf, dtype, queries):
    """More queries than cached tokens: the first ones lie before slot 0."""
    H, G, D = 2, 4, 64
    w = World(kvf, [(5, 0), (40, 0), (0, 0)], H, D, dtype, 16, seed=8)
    counts = [queries, queries, 3]
    b = w.cache.batch(w.seqs, counts, H * G)
    q = _randn((sum(counts), H * G, D), dtype, 3)
    out, lse = w.cache.attend(b, q, return_lse=True, decay=0.0)
    at = 0
    for i, c in enumerate(counts):
        n = w.lens[i][0]
        o, z, s, to, tz, ts = reference(w.k[i], w.v[i], q[at:at + c], 1 / 8, 0, 0, dtype)
        close(out[at:at + c], o, to)
        close(lse[at:at + c], z, tz)
        empty = max(0, c - n)
        assert (out[at:at + empty] == 0).all() and (lse[at:at + empty] == -math.inf).all()
        at += c


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("c", [4, 200])
def test_scores_of_minus_infinity(kvf, dtype, c):
    """A row whose every score is -inf is like a row that sees nothing; one
    finite score takes all the weight."""
    H, D = 1, 64
    w = World(kvf, [(130, c)], H, D, dtype, 16, seed=9)
    w.k[0].zero_()
    w.k[0][:, :, 0] = -math.inf
    w.k[0][-1] = 0.0
    q = torch.zeros((c, 2, D), dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    # 0 * inf would be NaN: the other channels of the keys are 0, as the query's
    b = w.cache.batch(w.seqs, [130])
    w.cache.append(b, w.k[0][:130], w.v[0][:130])
    w.step(2)
    out, lse = w.cache.attend(w.batch, q, return_lse=True)
    assert (out[:-1] == 0).all() and (lse[:-1] == -math.inf).all()
    assert torch.equal(out[-1], w.v[0][-1].expand(2, D)) and (lse[-1] == 0).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lens,window,sinks", [([(200, 3)], 0, 0), ([(100, 150)], 0, 0), ([(300, 180)], 64, 0),
                                               ([(400, 2)], 50, 4), ([(700, 260)], 130, 20)])
def test_nonfinite_values_in_hidden_places(kvf, dtype, bad, lens, window, sinks):
    """A non-finite value reaches exactly the rows that see it."""
    H, G, D = 2, 2, 64
    w = World(kvf, lens, H, D, dtype, 16, seed=10)
    n, c = sum(lens[0]), lens[0][1]
    for j in {n - 1, n - 1 - c // 2, n - c, 30, 7, max(0, n - c - window)}:
        w.v[0][j, 0, j % D] = bad
    old = lens[0][0]
    w.cache.append(w.cache.batch(w.seqs, [old]), w.k[0][:old], w.v[0][:old])
    check(w, w.step(H * G, window, sinks), window, sinks)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens,window", [([(100, 150)], 0), ([(300, 180)], 64), ([(200, 3)], 20)])
def test_nonfinite_keys_in_hidden_places(kvf, dtype, lens, window):
    H, G, D = 1, 2, 64
    w = World(kvf, lens, H, D, dtype, 16, seed=11)
    n, c = sum(lens[0]), lens[0][1]
    w.k[0][n - 1] = math.nan  # only the last token sees it
    if window:
        w.k[0][:n - c - window + 1] = math.inf  # nobody sees these
    old = lens[0][0]
    w.cache.append(w.cache.batch(w.seqs, [old]), w.k[0][:old], w.v[0][:old])
    q = w.step(H * G, window, 0)
    out, lse = w.cache.attend(w.batch, q, return_lse=True, decay=0.0)
    assert torch.isnan(out[-1]).all() and torch.isnan(lse[-1]).all()
    k, v = w.k[0].clone(), w.v[0]
    lo = max(0, n - c - window + 1) if window else 0
    k[n - 1] = 0.0
    k[:lo] = 0.0
    o, z, s, to, tz, ts = reference(k, v, q, 1 / 8, window, 0, dtype)
    close(out[:-1], o[:-1], to[:-1])
    close(lse[:-1], z[:-1], tz[:-1])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", [2, 5, 9, 14])
def test_weights_accumulate_and_decay(kvf, dtype, case):
    lens, H, G, D, page = SHAPES[case]
    w = World(kvf, lens, H, D, dtype, page, seed=case)
    q = w.step(H * G)
    before = []
    for i, seq in enumerate(w.seqs):
        pages = torch.tensor(w.cache.pages(seq), device="cuda", dtype=torch.long)
        n = sum(lens[i])
        x = torch.rand((H, len(pages) * page), generator=_gen(i), device="cuda")
        w.cache.weights[0, pages] = x.view(H, len(pages), page).transpose(0, 1)
        before.append(x[:, :n].clone())
    check(w, q, decay=0.75, before=before)
    # sequences without new tokens keep theirs
    for i, (seq, (a, c)) in enumerate(zip(w.seqs, lens)):
        if c == 0 and a:
            pages = torch.tensor(w.cache.pages(seq), device="cuda", dtype=torch.long)
            now = w.cache.weights[0, pages].transpose(0, 1).reshape(H, -1)[:, :a]
            assert torch.equal(now, before[i])


def test_new_tokens_start_without_weight(kvf):
    w = World(kvf, [(20, 5)], 2, 64, F16, 16, seed=1)
    pages = torch.tensor(w.cache.pages(w.seqs[0]), device="cuda", dtype=torch.long)
    w.step(4)
    x = w.cache.weights[0, pages].transpose(0, 1).reshape(2, -1)
    assert (x[:, :25] == 0).all() and torch.isnan(x[:, 25:]).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("case", [1, 6, 10, 14])
def test_the_same_bits_every_time(kvf, dtype, case):
    lens, H, G, D, page = SHAPES[case]
    w = World(kvf, lens, H, D, dtype, page, seed=case)
    q = w.step(H * G)
    first = w.cache.attend(w.batch, q, decay=0.0, return_lse=True) + (w.cache.weights.clone(),)
    for _ in range(3):
        again = w.cache.attend(w.batch, q, decay=0.0, return_lse=True) + (w.cache.weights,)
        for a, b in zip(first, again):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_strides(kvf, dtype):
    """Rows taken out of wider tensors, heads before tokens, an expanded query,
    and rows that start at odd elements."""
    H, G, D = 2, 4, 64
    for kind in ("wide", "transposed", "odd", "expanded"):
        w = World(kvf, [(70, 40), (20, 1)], H, D, dtype, 16, seed=12)
        q = w.step(H * G)
        n = q.shape[0]
        k = torch.cat([x[a:] for x, (a, _) in zip(w.k, w.lens)])
        if kind == "wide":
            box = torch.randn((n, H * G + 2 * H, D), device="cuda").to(dtype)
            box[:, :H * G] = q
            box[:, H * G:H * G + H] = k
            q2, k2 = box[:, :H * G], box[:, H * G:H * G + H]
        elif kind == "transposed":
            q2 = q.transpose(0, 1).contiguous().transpose(0, 1)
            k2 = k.transpose(0, 1).contiguous().transpose(0, 1)
        elif kind == "odd":
            box = torch.empty(n * H * G * (D + 1) + 1, device="cuda", dtype=dtype)
            q2 = box[1:].view(n, H * G, D + 1)[:, :, :D]
            q2.copy_(q)
            box = torch.empty(n * H * (D + 1) + 1, device="cuda", dtype=dtype)
            k2 = box[1:].view(n, H, D + 1)[:, :, :D]
            k2.copy_(k)
        else:
            q = q[:, :1].expand(n, H * G, D)
            q2, k2 = q, k
        v = torch.cat([x[a:] for x, (a, _) in zip(w.v, w.lens)])
        w.cache.append(w.batch, k2, v)
        a, b = w.cache.attend(w.batch, q.contiguous()), w.cache.attend(w.batch, q2)
        assert torch.equal(a, b), kind
        check(w, q2)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D,heads,group,lens", [(128, 2, 5, [(300, 100), (3, 1)]), (64, 1, 3, [(1000, 600)]),
                                                (128, 1, 150, [(200, 30), (64, 1)])])
def test_weights_of_strided_queries(kvf, dtype, D, heads, group, lens):
    """Rows that start at odd elements, or lie apart by odd strides, and more
    query heads per KV head than a tile has rows."""
    w = World(kvf, lens, heads, D, dtype, 32, seed=13)
    q = w.step(heads * group)
    n = q.shape[0]
    box = torch.empty(n * heads * group * (D + 1) + 1, device="cuda", dtype=dtype)
    q2 = box[1:].view(n, heads * group, D + 1)[:, :, :D]
    q2.copy_(q)
    check(w, q2, decay=0.0)
    wide = torch.zeros((n, heads * group, 2 * D), device="cuda", dtype=dtype)
    wide[:, :, D:] = q
    check(w, wide[:, :, D:], decay=0.0)
    one = q[:, :1].expand(n, heads * group, D)
    check(w, one, decay=0.0)


def test_other_streams(kvf):
    """Tokens appended on one stream are there for a call on another."""
    lens, H, G, D, page = SHAPES[14]
    w = World(kvf, lens, H, D, F16, page, seed=3)
    q = w.step(H * G)
    want = w.cache.attend(w.batch, q, decay=0.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    k = torch.cat([x[a:] for x, (a, _) in zip(w.k, lens)])
    v = torch.cat([x[a:] for x, (a, _) in zip(w.v, lens)])
    junk = torch.randn((4096, 4096), device="cuda")
    for i in range(6):
        with torch.cuda.stream(streams[i % 3]):
            for _ in range(10):  # the appending stream is busy
                junk @ junk
            w.cache.append(w.batch, -k if i < 5 else k, v)
        with torch.cuda.stream(streams[(i + 1) % 3]):
            b = w.cache.batch(w.seqs, [c for _, c in lens], H * G)
            got = w.cache.attend(b, q, decay=0.0)
            del b
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,dim", [(F16, 64), (BF16, 128), (F32, 20)])
def test_many_sequences(kvf, dtype, dim):
    """More sequences than multiprocessors by far, most of them shorter than a tile."""
    rng = np.random.RandomState(dim)
    lens = [(int(a), int(c)) for a, c in zip(rng.randint(0, 40, 2000), rng.randint(0, 3, 2000))]
    lens[7], lens[1500] = (900, 30), (0, 40)
    w = World(kvf, lens, 2, dim, dtype, 16, seed=dim)
    check(w, w.step(4), decay=0.0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_whole_prompt(kvf, dtype):
    w = World(kvf, [(0, 5001)], 1, 64, dtype, 64, seed=21)
    check(w, w.step(6, 3000, 5), 3000, 5, decay=0.0)


@pytest.mark.parametrize("dtype", [F32, F16])
def test_captured_step(kvf, dtype):
    """A step's calls in a CUDA graph, captured on the stream that the batch was
    made on, give the bits of the calls themselves, on new inputs too."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        w = World(kvf, [(200, 1), (30, 50)], 2, 64, dtype, 16, seed=22)
        q = w.step(8)
        n = q.shape[0]
        k = torch.cat([x[a:] for x, (a, _) in zip(w.k, w.lens)])
        v = torch.cat([x[a:] for x, (a, _) in zip(w.v, w.lens)])

        def step():
            w.cache.append(w.batch, k, v)
            return w.cache.attend(w.batch, q, decay=0.0, return_lse=True)

        step()
        graph = torch.cuda.CUDAGraph()
    s.synchronize()
    with torch.cuda.graph(graph, stream=s):
        out, lse = step()
    with torch.cuda.stream(s):
        for seed in (1, 2):
            for t in (q, k, v):
                t.copy_(_randn(t.shape, dtype, seed))
            w.cache.weights.fill_(9.0)
            graph.replay()
            got = out.clone(), lse.clone(), w.cache.weights.clone()
            w.cache.weights.fill_(9.0)
            want = step() + (w.cache.weights,)
            for a, b in zip(got, want):
                assert torch.equal(a, b)
    s.synchronize()


def test_layers_are_apart(kvf):
    w = World(kvf, [(40, 3)], 2, 64, F16, 16, layers=3, seed=4)
    q = w.step(4, layer=1)
    check(w, q, layer=1)
    assert torch.isnan(w.cache.attend(w.batch, q, layer=0)).any()  # its new tokens were not written


def test_cache_beyond_32_bits(kvf):
    """Pages behind 2^31 elements and 2^32 bytes of the pool."""
    H, D, page = 8, 128, 128
    P = 2 ** 31 // (H * D * page) + 300
    cache = kvf.PagedKVCache(P, H, D, page_size=page, dtype=F16)
    lens = [(1000, 1), (500, 200)]
    w = World.__new__(World)
    w.cache, w.lens, w.H, w.D, w.dtype = cache, lens, H, D, F16
    high = list(range(P - 1, P - 40, -1))
    w.seqs = [cache.add(0, pages=high[:10]), cache.add(0, pages=high[10:20])]
    w.k = [_randn((a + c, H, D), F16, i) for i, (a, c) in enumerate(lens)]
    w.v = [_randn((a + c, H, D), F16, i + 5) for i, (a, c) in enumerate(lens)]
    b = cache.extend(w.seqs, [a for a, _ in lens])
    cache.append(b, torch.cat([k[:a] for k, (a, _) in zip(w.k, lens)]),
                 torch.cat([v[:a] for v, (a, _) in zip(w.v, lens)]))
    check(w, w.step(32), decay=0.0)
    kv = cache.gather(w.seqs[1])
    assert torch.equal(kv.keys_tensor, w.k[1].transpose(0, 1))
    e = cache.evict(w.seqs, 100, recent=10, sinks=2)
    kv = cache.gather(e.seqs[0])
    kept = e.kept[0, 0].long()
    for h in range(H):
        assert torch.equal(kv.values_tensor[h], w.v[0][kept[h], h])


# ---- append, gather ------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [1, 7, 32, 80, 128, 200])
@pytest.mark.parametrize("page", [16, 128])
def test_append_and_gather(kvf, dtype, D, page):
    lens = [(0, 0), (1, 0), (page, 1), (page - 1, 2), (300, 0), (0, 40)]
    w = World(kvf, lens, 3, D, dtype, page, layers=2, seed=D)
    for layer in range(2):
        for i, (a, c) in enumerate(lens):
            kv = w.cache.gather(w.seqs[i], layer)
            assert kv.layer_idx == layer and kv.shape == (3, a, D)
            assert torch.equal(kv.keys_tensor, w.k[i][:a].transpose(0, 1))
            assert torch.equal(kv.values_tensor, w.v[i][:a].transpose(0, 1))
    w.step(3, layer=1)
    for i, (a, c) in enumerate(lens):
        kv = w.cache.gather(w.seqs[i], 1)
        assert torch.equal(kv.keys_tensor, w.k[i].transpose(0, 1))
        assert torch.equal(kv.values_tensor, w.v[i].transpose(0, 1))
    free = torch.ones(w.cache.num_pages, dtype=torch.bool)
    for s in w.seqs:
        free[w.cache.pages(s)] = False
    assert torch.isnan(w.cache.keys[1, free.cuda()]).all()  # nothing else was written


# ---- eviction --------------------------------------------------------------------------
def _kept(weight, n, budget, recent, sinks):
    """The kept slots of one head, from the definition: weight [n]."""
    if n <= budget:
        return list(range(n))
    always = [j for j in range(n) if j < sinks or j >= n - recent]
    rest = [j for j in range(n) if sinks <= j < n - recent]
    key = [(-math.inf, 0) if math.isnan(x) else (x, 1) for x in weight]
    rest.sort(key=lambda j: (-key[j][0], -key[j][1], j))
    return sorted(always + rest[:budget - len(always)])


@pytest.mark.parametrize("dtype,D", [(F16, 128), (F32, 20), (BF16, 65)])
@pytest.mark.parametrize("kind", ["random", "ties", "equal", "special", "tiny"])
@pytest.mark.parametrize("budget,recent,sinks", [(1, 0, 0), (100, 0, 0), (100, 100, 0), (100, 30, 5), (100, 0, 100),
                                                 (1500, 64, 4), (2049, 1000, 1)])
def test_evict(kvf, dtype, D, kind, budget, recent, sinks):
    page, H, Ls = 32, 3, 2
    lens = [2100, 1, 100, 101, 1499, 0, 2500]
    spare = sum(-(-min(n, budget) // page) for n in lens)
    w = World(kvf, [(n, 0) for n in lens], H, D, dtype, page, layers=Ls, seed=2, spare=spare)
    g = _gen(budget)
    wt = w.cache.weights
    shape = wt.shape
    if kind == "random":
        wt.copy_(torch.randn(shape, generator=g, device="cuda").exp())
    elif kind == "ties":
        wt.copy_(torch.randint(0, 4, shape, generator=g, device="cuda").float())
    elif kind == "equal":
        wt.fill_(0.25)
    elif kind == "special":
        pick = torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, 1e-42, -1e-42, 3.0, -3.0], device="cuda")
        wt.copy_(pick[torch.randint(0, len(pick), shape, generator=g, device="cuda")])
    else:  # values that differ in their last bits only
        wt.copy_(1.0 + torch.randint(0, 700, shape, generator=g, device="cuda").float() * 2.0 ** -23)
    old = []
    for i, s in enumerate(w.seqs):
        pages = torch.tensor(w.cache.pages(s), device="cuda", dtype=torch.long)
        old.append([x[:, pages].transpose(1, 2).reshape((Ls, H, -1) + x.shape[4:])[:, :, :lens[i]].clone()
                    for x in (w.cache.keys, w.cache.values, w.cache.weights)])
    free = w.cache.free_pages
    e = w.cache.evict(w.seqs, budget, recent, sinks)
    assert e.seqs == w.seqs and e.kept.shape == (Ls, len(lens), H, budget)
    kept = e.kept.cpu()
    used = sum(-(-n // page) for n in lens)
    assert w.cache.free_pages == free + used - spare
    for i, s in enumerate(w.seqs):
        m = min(budget, lens[i])
        assert w.cache.length(s) == m
        pages = torch.tensor(w.cache.pages(s), device="cuda", dtype=torch.long)
        new = [x[:, pages].transpose(1, 2).reshape((Ls, H, -1) + x.shape[4:])[:, :, :m]
               for x in (w.cache.keys, w.cache.values, w.cache.weights)]
        for layer in range(Ls):
            for h in range(H):
                k = kept[layer, i, h].tolist()
                want = _kept(old[i][2][layer, h].tolist(), lens[i], budget, recent, sinks)
                assert k[:m] == want and all(x == -1 for x in k[m:])
                for a, b in zip(new, old[i]):
                    assert torch.equal(a[layer, h].nan_to_num(9.0), b[layer, h, want].nan_to_num(9.0))


def test_evict_long_sequences(kvf):
    """More weights than the selection keeps in shared memory (200 KB), and page
    tables too long to travel with the launch."""
    page, H, lens = 32, 2, [52000, 70001, 30]
    budget, recent, sinks = 40000, 100, 4
    spare = sum(-(-min(n, budget) // page) for n in lens)
    w = World(kvf, [(n, 0) for n in lens], H, 8, F16, page, seed=6, spare=spare)
    wt = w.cache.weights
    wt.copy_(torch.randint(0, 50000, wt.shape, generator=_gen(8), device="cuda").float())
    old = []
    for s, n in zip(w.seqs, lens):
        pages = torch.tensor(w.cache.pages(s), device="cuda")
        old.append(wt[0, pages].transpose(0, 1).reshape(H, -1)[:, :n].cpu().tolist())
    e = w.cache.evict(w.seqs, budget, recent, sinks)
    kept = e.kept[0].cpu()
    for i, (s, n) in enumerate(zip(w.seqs, lens)):
        m = min(budget, n)
        kv = w.cache.gather(s)
        pages = torch.tensor(w.cache.pages(s), device="cuda")
        weights = w.cache.weights[0, pages].transpose(0, 1).reshape(H, -1)[:, :m].cpu()
        for h in range(H):
            want = _kept(old[i][h], n, budget, recent, sinks)
            assert kept[i, h, :m].tolist() == want and bool((kept[i, h, m:] == -1).all())
            at = torch.tensor(want, device="cuda")
            assert torch.equal(kv.keys_tensor[h], w.k[i][at, h]) and torch.equal(kv.values_tensor[h], w.v[i][at, h])
            assert weights[h].tolist() == [old[i][h][j] for j in want]


@pytest.mark.parametrize("dtype,D", [(F16, 64), (F32, 12)])
@pytest.mark.parametrize("n", [959 * 16, 960 * 16, 960 * 16 + 1, 1920 * 16 - 1, 1920 * 16 + 5])
def test_gather_of_many_pages(kvf, dtype, D, n):
    w = World(kvf, [(n, 0)], 2, D, dtype, 16, seed=n % 97)
    kv = w.cache.gather(w.seqs[0])
    assert torch.equal(kv.keys_tensor, w.k[0].transpose(0, 1))
    assert torch.equal(kv.values_tensor, w.v[0].transpose(0, 1))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("new,window,sinks", [(1, 0, 0), (1, 100001, 7), (40, 0, 0), (40, 70000, 130)])
def test_long_sequence(kvf, dtype, new, window, sinks):
    """150000 slots in 9375 pages, shared out over all multiprocessors, beside a
    short sequence."""
    w = World(kvf, [(150000 - new, new), (20, 1)], 1, 64, dtype, 16, seed=new)
    q = w.step(4, window, sinks)
    check(w, q, window, sinks, decay=0.0)


def test_evict_keeps_the_source(kvf):
    w = World(kvf, [(200, 0), (50, 0)], 2, 64, F16, 16, seed=5, spare=12)
    w.cache.weights.copy_(torch.rand(w.cache.weights.shape, generator=_gen(1), device="cuda"))
    before = [t.clone() for t in (w.cache.keys, w.cache.values, w.cache.weights)]
    pages = [w.cache.pages(s) for s in w.seqs]
    e = w.cache.evict(w.seqs, 80, recent=8, sinks=2, keep_source=True)
    assert set(e.seqs).isdisjoint(w.seqs) and [w.cache.length(s) for s in e.seqs] == [80, 50]
    assert [w.cache.pages(s) for s in w.seqs] == pages and [w.cache.length(s) for s in w.seqs] == [200, 50]
    own = torch.tensor(sum(pages, []), device="cuda")
    for t, b in zip((w.cache.keys, w.cache.values, w.cache.weights), before):
        assert torch.equal(t[:, own].nan_to_num(3.0), b[:, own].nan_to_num(3.0))
    # the branch goes on by itself
    k = _randn((3, 2, 64), F16, 1)
    b = w.cache.extend(e.seqs, [2, 1], 4)
    w.cache.append(b, k, k)
    out = w.cache.attend(b, _randn((3, 4, 64), F16, 2))
    assert torch.isfinite(out).all()
    free = w.cache.free_pages
    w.cache.free(e.seqs)
    assert w.cache.free_pages == free + 5 + 1 + 4


def test_append_attend_evict_compress(kvf, oracle):
    """The operators together: a prompt, single tokens, an eviction, more tokens,
    and the codec at the end."""
    H, G, D = 2, 4, 128
    cache = kvf.PagedKVCache(40, H, D, page_size=32, dtype=F16)
    s = cache.add()

    def step(c, seed):
        k, v = _randn((c, H, D), F16, seed), _randn((c, H, D), F16, seed + 1)
        q = _randn((c, H * G, D), F16, seed + 2)
        b = cache.extend([s], [c], H * G)
        cache.append(b, k, v)
        return cache.attend(b, q, decay=1.0), k, v, q

    total = torch.zeros((H, 0), dtype=torch.float64, device="cuda")
    K = V = None
    for i, c in enumerate([300, 1, 1, 40, 1]):
        out, k, v, q = step(c, 10 * i)
        K = k if K is None else torch.cat([K, k])
        V = v if V is None else torch.cat([V, v])
        o, _, ws, to, _, _ = reference(K, V, q, D ** -0.5, 0, 0, F16)
        close(out, o, to)
        total = torch.cat([total, torch.zeros((H, c), dtype=torch.float64, device="cuda")], 1) + ws
    e = cache.evict([s], 120, recent=20, sinks=4)
    kept = e.kept[0, 0].long()
    for h in range(H):
        assert kept[h, :4].tolist() == [0, 1, 2, 3] and kept[h, -20:].tolist() == list(range(323, 343))
        mid, rest = kept[h, 4:-20], torch.ones(343, dtype=torch.bool, device="cuda")
        rest[kept[h]] = False
        assert total[h, mid].min() >= total[h, rest].max() * (1 - 1e-5)
    K = torch.stack([K[kept[h], h] for h in range(H)], 1)
    V = torch.stack([V[kept[h], h] for h in range(H)], 1)
    out, k, v, q = step(5, 777)
    K, V = torch.cat([K, k]), torch.cat([V, v])
    o, _, _, to, _, _ = reference(K, V, q, D ** -0.5, 0, 0, F16)
    close(out, o, to)
    kv = cache.gather(s)
    assert torch.equal(kv.keys_tensor, K.transpose(0, 1))
    c = kvf.compress(kv, "conservative")
    co = oracle.compress(kv.keys(), kv.values(), "conservative", 0, None, threads=2)
    assert c.ratio() == oracle.ratio(co)


# ---- refusals -----------------------------------------------------------------------------
def test_refusals(kvf):
    from kvforge_b200 import _lib as L
    err = kvf.KvForgeError
    with pytest.raises(TypeError):
        kvf.PagedKVCache(4, 1, 64, dtype=torch.float64)
    for bad in (dict(page_size=24), dict(page_size=8), dict(head_dim=0), dict(head_dim=257), dict(num_pages=0),
                dict(num_layers=0)):
        with pytest.raises(err):
            kvf.PagedKVCache(**{**dict(num_pages=4, num_heads=1, head_dim=64), **bad})
    c = kvf.PagedKVCache(6, 2, 64, page_size=16)
    s = c.add(20)
    with pytest.raises(err):
        c.add(200)  # not enough pages
    with pytest.raises(err):
        c.add(20, pages=[5])  # too few
    with pytest.raises(err):
        c.add(5, pages=[0])  # in use
    with pytest.raises(err):
        c.add(20, pages=[4, 4])
    with pytest.raises(err):
        c.extend([s], [1000], 4)
    assert c.length(s) == 20 and c.free_pages == 4
    for seqs, new, kw in (([s, s], [1, 1], {}), ([s], [1, 2], {}), ([s], [-1], {}), ([99], [1], {}),
                          ([s], [1], dict(query_heads=3)), ([s], [1], dict(query_heads=4, window=-1)),
                          ([s], [1], dict(query_heads=4, window=3, sinks=-1))):
        with pytest.raises(err):
            c.extend(seqs, new, **kw)
        assert c.length(s) == 20
    b = c.extend([s], [2], 4)
    q = torch.zeros((2, 4, 64), dtype=F16, device="cuda")
    k = torch.zeros((2, 2, 64), dtype=F16, device="cuda")
    for bad in (q.float(), q.bfloat16()):
        with pytest.raises(TypeError):
            c.attend(b, bad)
    for bad in (q[:1], q[:, :2], q[:, :, :32], q.cpu()):
        with pytest.raises(err):
            c.attend(b, bad)
    for kw in (dict(layer=1), dict(layer=-1), dict(scale=math.nan), dict(scale=math.inf), dict(decay=1.5),
               dict(decay=-0.5), dict(decay=math.nan)):
        with pytest.raises(err):
            c.attend(b, q, **kw)
    with pytest.raises(err):
        c.attend(c.batch([s], [2]), q)  # made without query heads
    with pytest.raises(err):
        c.append(b, k, k[:1])
    with pytest.raises(TypeError):
        c.append(b, k, k.float())
    for kw in (dict(budget=0), dict(budget=5, recent=4, sinks=2), dict(budget=5, recent=-1), dict(budget=5, sinks=-1)):
        with pytest.raises(err):
            c.evict([s], **kw)
    full = c.add(64)
    with pytest.raises(err):
        c.evict([s], 10)  # no free page to move to
    assert c.length(s) == 22
    c.free(full)
    c.evict([s], 10)
    with pytest.raises(err):
        c.append(b, k, k)  # its sequence was evicted since
    with pytest.raises(err):
        c.gather(full)
    # the C entry points by themselves
    lib, ctx = L.lib(), L.context(0)
    plan = C.c_void_p()
    i32 = lambda *x: np.array(x, np.int32)  # noqa: E731
    one, tab = i32(1), i32(0)
    make = lambda q=one, kv=one, t=tab, stride=1, qh=2, w=0, sk=0, pool=c._pool: lib.kvf_paged_plan_create(  # noqa: E731
        ctx, C.byref(pool), 1, q.ctypes.data, kv.ctypes.data, t.ctypes.data, stride, qh, w, sk, C.byref(plan), None)
    assert make(t=i32(6)) == L.ERR_SHAPE_MISMATCH and make(t=i32(-1)) == L.ERR_SHAPE_MISMATCH
    assert make(kv=i32(17)) == L.ERR_SHAPE_MISMATCH and make(kv=i32(-1)) == L.ERR_SHAPE_MISMATCH
    assert make(q=i32(-1)) == L.ERR_SHAPE_MISMATCH and make(qh=3) == L.ERR_SHAPE_MISMATCH
    assert make(w=-1) == L.ERR_INVALID_CONFIG and plan.value is None
    other = L.PagedPool.from_buffer_copy(c._pool)
    other.keys += 2
    assert make(pool=other) == L.ERR_INVALID_CONFIG
    assert make() == L.OK
    other = L.PagedPool.from_buffer_copy(c._pool)
    other.num_heads = 1
    assert lib.kvf_paged_append(ctx, plan, C.byref(other), 0, k.data_ptr(), 64, 64, k.data_ptr(), 64, 64,
                                None) == L.ERR_SHAPE_MISMATCH
    assert lib.kvf_paged_append(ctx, plan, C.byref(c._pool), 0, None, 64, 64, None, 64, 64, None) == L.ERR_INVALID_CONFIG
    other = L.PagedPool.from_buffer_copy(c._pool)
    other.weights = None
    assert lib.kvf_paged_attention(ctx, plan, C.byref(other), 0, q.data_ptr(), 256, 64, 1.0, 0.0, q.data_ptr(), None,
                                   None) == L.ERR_INVALID_CONFIG
    kept = torch.empty(1024, dtype=torch.int32, device="cuda")
    evict = lambda new, pool=c._pool, kv=one, t=tab, stride=1, n=1: lib.kvf_paged_evict(  # noqa: E731
        ctx, C.byref(pool), n, kv.ctypes.data, t.ctypes.data, stride, 1, 0, 0, new.ctypes.data, 1, kept.data_ptr(),
        None)
    assert evict(i32(0)) == L.ERR_INVALID_CONFIG  # the source's own page
    assert evict(i32(1), pool=other) == L.ERR_INVALID_CONFIG  # no weights
    assert evict(i32(6)) == L.ERR_SHAPE_MISMATCH and evict(i32(1), t=i32(-1)) == L.ERR_SHAPE_MISMATCH
    assert evict(i32(1), kv=i32(17)) == L.ERR_SHAPE_MISMATCH and evict(i32(1), kv=i32(-1)) == L.ERR_SHAPE_MISMATCH
    assert evict(i32(2, 2), kv=i32(1, 1), t=i32(0, 1), n=2) == L.ERR_INVALID_CONFIG  # named twice
    assert lib.kvf_paged_gather(ctx, C.byref(c._pool), 1, tab.ctypes.data, 1, k.data_ptr(), k.data_ptr(),
                                None) == L.ERR_SHAPE_MISMATCH
    assert lib.kvf_paged_gather(ctx, C.byref(c._pool), 0, i32(6).ctypes.data, 1, k.data_ptr(), k.data_ptr(),
                                None) == L.ERR_SHAPE_MISMATCH
    assert lib.kvf_paged_plan_free(plan) == L.OK and lib.kvf_paged_plan_free(None) == L.OK
    # the codec's entry points do not take bf16
    x = torch.zeros((1, 64, 64), dtype=BF16, device="cuda")
    assert lib.kvf_calibrate(ctx, x.data_ptr(), L.IN_BF16, 1, 64, 64, 1, kept.data_ptr(), None) == L.ERR_INVALID_CONFIG


def test_empty_calls(kvf):
    c = kvf.PagedKVCache(4, 2, 64, page_size=16)
    s = c.add()
    b = c.extend([s], [0], 4)
    none = torch.empty((0, 2, 64), dtype=F16, device="cuda")
    c.append(b, none, none)
    assert c.attend(b, torch.empty((0, 4, 64), dtype=F16, device="cuda"), decay=0.5).shape == (0, 4, 64)
    assert c.gather(s).shape == (2, 0, 64)
    e = c.evict([s], 3)
    assert (e.kept == -1).all() and c.length(s) == 0
    b = c.extend([], [], 4)
    assert b.tokens == 0 and c.evict([], 3).seqs == []


def test_example_runs():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, "examples", "paged_cache.py"), "--tokens", "700", "--budget",
                        "300", "--layers", "2"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    assert "evicted to 300 tokens" in r.stdout and "layer 1:" in r.stdout


# ---- rows, batches and calls out of the ordinary ------------------------------------------
@pytest.mark.parametrize("D", [20, 64, 100, 128, 200, 256])
@pytest.mark.parametrize("queries", [4, 16, 100, 900])
def test_rows_of_a_tile_without_slots_then_others(kvf, D, queries):
    """f32, whose rows are copied asynchronously: many tiles of rows that see
    nothing, each followed by tiles that see slots, in one CTA's share."""
    H, G, n = 2, 4, 24
    lens = [(7, 0), (90, 3)] * n
    w = World(kvf, lens, H, D, F32, 16, seed=D)
    w.step(H * G)
    counts = [queries, 3] * n
    b = w.cache.batch(w.seqs, counts, H * G)
    q = _randn((sum(counts), H * G, D), F32, 3)
    first = w.cache.attend(b, q, return_lse=True, decay=0.0)
    at = 0
    for i, c in enumerate(counts):
        if i < 4 or i >= 2 * n - 4:
            o, z, _, to, tz, _ = reference(w.k[i], w.v[i], q[at:at + c], D ** -0.5, 0, 0, F32)
            close(first[0][at:at + c], o, to, f"out of sequence {i}")
            close(first[1][at:at + c], z, tz, f"lse of sequence {i}")
        at += c
    for _ in range(5):
        for x, y in zip(first, w.cache.attend(b, q, return_lse=True, decay=0.0)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype,D", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("c,window,sinks", [(1, 0, 0), (4, 0, 0), (2, 40, 3), (1, 65, 70)])
def test_tiles_put_right_and_loaded_over(kvf, dtype, D, c, window, sinks):
    """Many short sequences whose tiles all have masked slots: values that are
    replaced in shared memory (the pages around them hold NaN) and the next tiles
    that arrive in the same place, without a trace of one in the other."""
    rng = np.random.RandomState(D + c)
    lens = [(int(a), c) for a in rng.randint(0, 140, 160)]
    w = World(kvf, lens, 4, D, dtype, 16, seed=c + window)
    q = w.step(16, window, sinks)
    first = check(w, q, window, sinks)
    for _ in range(10):
        for x, y in zip(first, w.cache.attend(w.batch, q, return_lse=True)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", [1, 4, 6, 10, 14])
def test_weights_of_queries_in_turn(kvf, dtype, case):
    """Calls of one batch share scores and parts of sums: each call's weights are
    its own queries', right behind those of others."""
    lens, H, G, D, page = SHAPES[case]
    w = World(kvf, lens, H, D, dtype, page, seed=case)
    w.cache.weights.zero_()
    qs = [w.step(H * G)] + [_randn((w.batch.tokens, H * G, D), dtype, 50 + i) for i in range(2)]
    want = []
    for q in qs:
        check(w, q, decay=0.0)
        want.append(w.cache.weights.clone())
    got = []
    for i in range(30):
        w.cache.attend(w.batch, qs[i % 3], decay=0.0)
        got.append(w.cache.weights.clone())
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 3]), i


@pytest.mark.parametrize("dtype,D", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("singles", [1, 9, 30])
def test_infinite_values_of_long_and_short_rows_in_turn(kvf, dtype, D, singles):
    """Shares of many segments, of one and of two row tiles: an infinite value
    reaches its own sequence's rows that see it, and no others. All other values
    are 1, so that an output is 1 to within the numerators' and its own rounding
    (u each) and the f32 sums' (less than u)."""
    H, G = 8, 4
    lens = ([(10, 45)] + [(5, 6 + i % 20) for i in range(singles)]) * (200 // (singles + 1))
    w = World(kvf, lens, H, D, dtype, 16, seed=singles)
    rng = np.random.RandomState(singles)
    want, at = [], 0
    for i, (a, c) in enumerate(lens):
        w.v[i].fill_(1.0)
        inf = torch.zeros((c, H, D), dtype=torch.bool, device="cuda")
        if i % 3 != 1:
            j, h, col = int(rng.randint(a, a + c)), int(rng.randint(H)), int(rng.randint(D))
            w.v[i][j, h, col] = math.inf
            inf[j - a:, h, col] = True  # the rows from its own token on
        want.append(inf.repeat_interleave(G, 1))
    old = w.cache.batch(w.seqs, [a for a, _ in lens])
    w.cache.append(old, torch.cat([k[:a] for k, (a, _) in zip(w.k, lens)]),
                   torch.cat([v[:a] for v, (a, _) in zip(w.v, lens)]))
    q, want = w.step(H * G), torch.cat(want)
    for _ in range(5):
        out = w.cache.attend(w.batch, q)
        assert torch.equal(torch.isinf(out), want)
        assert (out[~want].double() - 1.0).abs().max() <= 3 * UNIT[dtype]


@pytest.mark.parametrize("dtype", [F32, F16])
def test_captured_step_after_a_call_that_took_the_lse(kvf, dtype):
    """The workspace of the first call with decay serves every later one: a graph
    of calls without lse, replayed between calls of their own."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        w = World(kvf, [(200, 1), (30, 50)], 2, 64, dtype, 16, seed=22)
        q = w.step(8)
        w.cache.weights.fill_(0.0)
        w.cache.attend(w.batch, q, decay=0.0, return_lse=True)
        want_w = w.cache.weights.clone()
        graph = torch.cuda.CUDAGraph()
    s.synchronize()
    with torch.cuda.graph(graph, stream=s):
        out = w.cache.attend(w.batch, q, decay=0.0)
    with torch.cuda.stream(s):
        want = w.cache.attend(w.batch, q, decay=0.0)
        live = torch.tensor(sum((w.cache.pages(x) for x in w.seqs), []), device="cuda")
        for _ in range(3):
            w.cache.weights.fill_(9.0)
            out.fill_(9.0)
            graph.replay()
            a, b = w.cache.weights[:, live], want_w[:, live]
            assert torch.equal(out, want) and torch.equal(w.cache.attend(w.batch, q, decay=0.0), want)
            assert torch.equal(a[a != 9.0], b[a != 9.0]) and (a != 9.0).sum() == 2 * 281
    s.synchronize()
    del graph


def test_what_a_capture_refuses(kvf):
    """A batch, the first call with decay, and an eviction with long tables keep
    memory or read buffers that a graph must not hold: errors, lengths as before."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        w = World(kvf, [(200, 1), (30, 50), (20000, 0)], 2, 64, F16, 16, seed=23, spare=20)
        q = w.step(8)
        want = w.cache.attend(w.batch, q)
        graph = torch.cuda.CUDAGraph()
        lengths, free = [w.cache.length(x) for x in w.seqs], w.cache.free_pages
    s.synchronize()
    with torch.cuda.graph(graph, stream=s):
        for call in (lambda: w.cache.extend(w.seqs, [1, 1, 1], 8), lambda: w.cache.batch(w.seqs, [1, 1, 1], 8),
                     lambda: w.cache.attend(w.batch, q, decay=1.0),
                     lambda: w.cache.attend(w.batch, q, decay=1.0, return_lse=True),
                     lambda: w.cache.evict(w.seqs[2], 100)):
            with pytest.raises(kvf.KvForgeError, match="capture"):
                call()
        out = w.cache.attend(w.batch, q)
    assert [w.cache.length(x) for x in w.seqs] == lengths and w.cache.free_pages <= free
    with torch.cuda.stream(s):
        graph.replay()
        assert torch.equal(out, want)
        check(w, q, decay=0.0)
    s.synchronize()
    del graph


def _attend_into(w, b, q, value):
    """kvf_paged_attention on outputs that hold `value` before the call."""
    from kvforge_b200 import _lib as L
    out, lse = torch.full_like(q, value), torch.full(q.shape[:2], value, dtype=F32, device="cuda")
    L.check(L.lib().kvf_paged_attention(
        L.context(0), b._h, C.byref(w.cache._pool), 0, q.data_ptr(), q.stride(0), q.stride(1),
        w.D ** -0.5, -1.0, out.data_ptr(), lse.data_ptr(),
        torch.cuda.current_stream().cuda_stream))
    return out, lse


@pytest.mark.parametrize("dtype,D", [(F32, 64), (F32, 128), (F32, 200), (F16, 20), (BF16, 36), (F16, 64), (BF16, 128)])
@pytest.mark.parametrize("queries", [3, 70, 300])
@pytest.mark.parametrize("beside", [None, (9, 1), (400, 90)])
def test_queries_of_empty_sequences(kvf, dtype, D, queries, beside):
    """Sequences without any slot, alone or beside others: every row is written."""
    H, G = 2, 4
    lens = [(0, 0), (0, 0)] + ([beside] if beside else [])
    w = World(kvf, lens, H, D, dtype, 16, seed=queries)
    if beside:
        w.step(H * G)
    counts = [queries, queries + 1] + ([beside[1]] if beside else [])
    b = w.cache.batch(w.seqs, counts, H * G)
    q = _randn((sum(counts), H * G, D), dtype, 3)
    out, lse = _attend_into(w, b, q, math.nan)
    empty = 2 * queries + 1
    assert (out[:empty] == 0).all() and (lse[:empty] == -math.inf).all()
    if beside:
        o, z, _, to, tz, _ = reference(w.k[2], w.v[2], q[empty:], D ** -0.5, 0, 0, dtype)
        close(out[empty:], o, to)
        close(lse[empty:], z, tz)


def test_two_host_threads(kvf):
    """Two caches, each with a thread and a stream of its own, whose calls launch
    the same kernels with different amounts of shared memory."""
    import threading
    from kvforge_b200 import _lib as L
    lib, ctx, caches, fail = L.lib(), L.context(0), [], []
    for n, D in ((9000, 136), (30000, 256)):
        w = World(kvf, [(n, 0), (3, 1)], 1, D, F32, 128, seed=D)
        w.cache.weights.fill_(1.0)
        caches.append(w)
    torch.cuda.synchronize()
    go = threading.Barrier(2)

    def work(w):
        c = w.cache
        with torch.cuda.stream(torch.cuda.Stream()):
            b = c.extend(w.seqs[1:], [1], 2)
            q = torch.ones((1, 2, w.D), device="cuda")
            out, kept = torch.empty_like(q), torch.empty(50, dtype=torch.int32, device="cuda")
            st = torch.cuda.current_stream().cuda_stream
            pool, scale = C.byref(c._pool), C.c_float(1.0)
            pages = np.array(c.pages(w.seqs[0]), np.int32)
            lens, new = np.array([w.lens[0][0]], np.int32), np.array(c._free[:1], np.int32)
            go.wait()
            for i in range(20000):
                r = lib.kvf_paged_attention(ctx, b._h, pool, 0, q.data_ptr(), 2 * w.D, w.D, scale, 0.0, out.data_ptr(),
                                            None, st)
                if r == 0 and i % 20 == 0:
                    r = lib.kvf_paged_evict(ctx, pool, 1, lens.ctypes.data, pages.ctypes.data, len(pages), 50, 0, 0,
                                            new.ctypes.data, 1, kept.data_ptr(), st)
                if r:
                    fail.append((i, lib.kvf_last_error()))
                    return

    threads = [threading.Thread(target=work, args=(c,)) for c in caches]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not fail, fail


def test_batch_of_another_cache(kvf):
    """A batch names pages of its own cache: another one of the same shape refuses it."""
    a, b = (kvf.PagedKVCache(8, 2, 64, page_size=16) for _ in range(2))
    batch = a.extend([a.add()], [3], 4)
    b.extend([b.add()], [3], 4)
    k, q = _randn((3, 2, 64), F16, 1), _randn((3, 4, 64), F16, 2)
    for call in (lambda: b.append(batch, k, k), lambda: b.attend(batch, q), lambda: b.attend(batch, q, decay=0.0)):
        with pytest.raises(kvf.KvForgeError, match="another cache"):
            call()
    assert not b.keys.any() and not b.values.any() and not b.weights.any()
    a.append(batch, k, k)
    assert torch.isfinite(a.attend(batch, q)).all()


def test_a_wait_that_gave_up_is_told(kvf):
    """A bounded device wait that runs out (the library's self-test of one) is told
    by sync, once, and the cache goes on."""
    from kvforge_b200 import _lib as L
    w = World(kvf, [(40, 1), (7, 30)], 2, 64, F16, 16, seed=31)
    q = w.step(4)
    w.cache.sync()
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    L.check(L.lib().kvf_selftest_wait_timeout(L.context(0), L.WAIT_MBARRIER, st))
    w.cache.attend(w.batch, q)
    with pytest.raises(kvf.KvForgeError) as e:
        w.cache.sync()
    assert e.value.status == L.ERR_DEVICE_TIMEOUT
    w.cache.sync()
    check(w, q, decay=0.0)
    w.cache.sync()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("lens,row", [((100, 4), 1), ((500, 7), 0), ((3, 2), 0), ((200, 60), 20)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2), (70, 0)])
def test_weights_of_a_nan_row(kvf, dtype, lens, row, window, sinks):
    """A query of NaN gives NaN weights to the slots that it sees, and to no others."""
    H, G, D = 2, 2, 64
    w = World(kvf, [lens], H, D, dtype, 16, seed=40)
    q = w.step(H * G, window, sinks)
    bad = q.clone()
    bad[row, 1] = math.nan  # KV head 0
    w.cache.attend(w.batch, bad, decay=0.0)
    (a, c), n = lens, sum(lens)
    pages = torch.tensor(w.cache.pages(w.seqs[0]), device="cuda")
    got = w.cache.weights[0, pages].transpose(0, 1).reshape(H, -1)[:, :n]
    _, _, want, _, _, tol = reference(w.k[0], w.v[0], q, D ** -0.5, window, sinks, dtype)
    see = seen(n, c, window, sinks)[row]
    s = (w.k[0][:, 0].double() @ q[row, 1].double() * D ** -0.5).masked_fill(~see, -math.inf)
    want[0] -= torch.softmax(s, 0)
    want[0, see] = math.nan
    close(got, want, tol + 2.0 ** -40)


def test_evict_without_memory_for_its_result(kvf):
    """A budget whose list of kept slots (2^48 bytes) fits nowhere: an error, and no page is lost."""
    cache = kvf.PagedKVCache(8, 16, 8, page_size=16, num_layers=4096)
    s = cache.add(40)
    free = cache.free_pages
    with pytest.raises(RuntimeError):
        cache.evict([s], 2 ** 30)
    assert cache.free_pages == free and cache.length(s) == 40
    cache.evict([s], 20)
    assert cache.free_pages == free + 1 and cache.length(s) == 20


@pytest.mark.parametrize("window,sinks", [(2 ** 31, 0), (2 ** 32 + 5, 0), (2 ** 70, 3), (7, 2 ** 32), (7, 2 ** 32 + 3)])
def test_windows_beyond_32_bits(kvf, window, sinks):
    """A window, or sinks, longer than any sequence hides nothing."""
    w = World(kvf, [(300, 1), (50, 70)], 2, 64, F16, 16, seed=41)
    check(w, w.step(4, window, sinks), decay=0.0)
    for bad in (dict(window=-2 ** 32), dict(window=9, sinks=-2 ** 32)):
        with pytest.raises(kvf.KvForgeError):
            w.cache.batch(w.seqs, [1, 1], 4, **bad)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [0.0, -0.0, 0.3, -0.3])
def test_nan_queries_at_any_scale(kvf, dtype, scale):
    """A NaN query gives NaN, also where the scale is 0; the other rows are as ever."""
    w = World(kvf, [(300, 1), (50, 70), (9, 3)], 2, 64, dtype, 32, seed=42, big=30.0)
    for i in range(3):
        w.cache.append(w.cache.batch(w.seqs[i:i + 1], [w.lens[i][0]]), w.k[i][:w.lens[i][0]], w.v[i][:w.lens[i][0]])
    q = w.step(8) * 30
    want, want_lse = check(w, q, scale=scale)
    bad = q.clone()
    hit = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    for t, h in ((0, 3), (5, 0), (40, 7), (72, 2)):
        bad[t, h, 11], hit[t, h] = math.nan, True
    out, lse = w.cache.attend(w.batch, bad, scale=scale, return_lse=True)
    assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
    assert torch.equal(out[~hit], want[~hit]) and torch.equal(lse[~hit], want_lse[~hit])


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale", [0.0, 1e-44, -1e-40, 1e-38, 1e-30])
def test_vanishing_scales_under_a_window(kvf, dtype, scale):
    """Rows whose first tiles are all masked, at scales that make every score the same."""
    w = World(kvf, [(152, 237), (600, 300), (90, 2)], 2, 64, dtype, 32, seed=43)
    check(w, w.step(2, 1, 0), 1, 0, scale=scale, decay=0.0)
    b = w.cache.batch(w.seqs, [c for _, c in w.lens], 2, 41, 3)
    w.batch = b
    check(w, _randn((b.tokens, 2, 64), dtype, 9), 41, 3, scale=scale, decay=0.0)
