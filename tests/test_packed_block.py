"""The operators of a block over packed rows -- packed_attention, projection,
block_norm -- against plain implementations in 64 bits, their refusals, and a
block run through all of them.

Tolerances.  u is half a step of the output's type relative to its value
(fp16 2^-11, bf16 2^-8, fp32 2^-24), e = 2^-24 that of the fp32 arithmetic.
  attention   The weights p are rounded to the type, for P.V and for their
              sum: with p (1 + r), |r| <= u, the output moves by sum r p (v -
              out) / sum p, at most u (sum p|v| / sum p + |out|) (fp16 also by
              2^-25 (|v| + |out|) a key below its normal range, with the
              largest p at least 1), and by u |out| (and 2^-25) when it is
              rounded itself.  A score of D products moves by
              d = (D + 8) e scale sum|q k|, a weight by twice that of the
              worst key and 2^-20 for the exponential, the sums by n e.
  projection  (k + 8) e sum|x w| before the activation, whose slope is at most
              1.13, 2^-15 |act| for the activation itself, u |out|, and 4 e of
              the epilogue's terms.
  block_norm  2^-18 of the largest normed entry of a row (sums of up to 32,768
              terms in a tree of 16 or more partial sums of 64 lanes, each
              within 64 e, and the cancellation in x - mean), twice for the
              second norm, whose input also moves by the first's error over
              its own spread; u |out|.
"""

import ctypes as C
import math

import numpy as np
import pytest
import torch

from gliner_decide import _native as N

gpu = pytest.mark.gpu
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
E = 2.0 ** -24
FAKE = 0x10000  # never dereferenced: validation fails before any launch


def fk():
    from gliner_decide.fused_kernels import FusedKernels
    return FusedKernels()


def normal(seed, *shape, dtype=torch.float16, scale=1.0, mean=0.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.empty(shape, device="cuda").normal_(mean, scale, generator=g).to(dtype)


def offsets(lengths, dtype=torch.int32):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64), dtype=dtype, device="cuda")


def within(got, want, tol, what=""):
    torch.cuda.synchronize()
    diff = (got.double() - want).abs()
    bad = ~(diff <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(diff[bad].max()):.3g} "
                           f"with {float(tol[bad].min()):.3g} allowed")


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def attention_reference(q, k, v, q_lengths, k_lengths, scale, causal):
    """(out, tolerance) in 64 bits, one sequence and head at a time."""
    Tq, H, D = q.shape
    group = H // k.shape[1]
    u = HALF_STEP[q.dtype]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    q0 = k0 = 0
    for nq, nk in zip(q_lengths, k_lengths):
        for h in range(H):
            qq = q[q0:q0 + nq, h].double()
            kk, vv = k[k0:k0 + nk, h // group].double(), v[k0:k0 + nk, h // group].double()
            if nq == 0 or nk == 0:
                continue
            s = (qq @ kk.T.contiguous()) * scale
            mag = (qq.abs() @ kk.abs().T.contiguous()) * abs(scale)
            if causal:
                hidden = torch.arange(nk, device=q.device)[None] > torch.arange(nq, device=q.device)[:, None] + nk - nq
                s = s.masked_fill(hidden, -math.inf)
                mag = mag.masked_fill(hidden, 0.0)
            some = ~torch.isinf(s).all(-1, keepdim=True)
            top = torch.where(some, s.amax(-1, keepdim=True), 0.0)
            p = torch.exp(s - top)
            total = p.sum(-1, keepdim=True).clamp(min=1e-300)
            o = (p @ vv) / total
            av = (p @ vv.abs()) / total
            d = (D + 8) * E * mag.amax(-1, keepdim=True)
            t = 2 * u * o.abs() + TINY[q.dtype] + av * (u + 2 * d + 2.0 ** -20 + nk * E)
            if q.dtype == torch.float16:
                visible = (~torch.isinf(s)).double()
                t = t + 2.0 ** -25 * (visible @ vv.abs() + visible.sum(-1, keepdim=True) * o.abs())
            out[q0:q0 + nq, h] = torch.where(some, o, 0.0)
            tol[q0:q0 + nq, h] = torch.where(some, t, 0.0)
        q0 += nq
        k0 += nk
    return out, tol


def check_attention(q, k, v, q_lengths, k_lengths, causal=True, scale=None):
    """k_lengths None: the queries' own tokens."""
    got = fk().packed_attention(q, k, v, offsets(q_lengths), None if k_lengths is None else offsets(k_lengths),
                                causal=causal, scale=scale)
    assert got.shape == q.shape and got.dtype == q.dtype
    want, tol = attention_reference(q, k, v, q_lengths, q_lengths if k_lengths is None else k_lengths,
                                    q.shape[2] ** -0.5 if scale is None else scale, causal)
    within(got, want, tol, "attention")
    return got


LENGTHS = [
    ([1], None),
    ([64], None),
    ([1, 0, 2, 15, 16, 17], None),
    ([31, 32, 33, 63, 65], None),
    ([127, 128, 129, 1, 255, 257], None),
    ([700, 3], None),
    ([1], [1]),
    ([1], [513]),
    ([1, 1, 1], [1, 0, 4097]),
    ([1] * 70, list(range(1, 71))),
    ([5, 1, 0, 3], [5, 33, 7, 300]),
    ([130, 1, 64], [1000, 2049, 64]),
    ([20, 300, 3], [3, 40, 0]),  # more queries than keys: the first see none under the causal order
    ([2, 2], [6000, 1]),
    ([200], [5000]),
]


@gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (16, 4, 64), (8, 1, 128), (15, 3, 128), (6, 2, 32),
                                                (5, 1, 96), (4, 2, 192), (8, 2, 256), (40, 2, 64)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_lengths(dtype, heads, kv_heads, dim, causal):
    for i, (ql, kl) in enumerate(LENGTHS):
        q = normal(10 * i, sum(ql), heads, dim, dtype=dtype)
        tk = sum(ql if kl is None else kl)
        k, v = normal(10 * i + 1, tk, kv_heads, dim, dtype=dtype), normal(10 * i + 2, tk, kv_heads, dim, dtype=dtype)
        check_attention(q, k, v, ql, kl, causal)


@gpu
@pytest.mark.parametrize("seed", range(12))
def test_attention_drawn_lengths(seed):
    r = np.random.default_rng(seed)
    for _ in range(4):
        kv_heads = int(r.choice([1, 2, 3]))
        heads = kv_heads * int(r.choice([1, 2, 3, 7, 8]))
        dim = int(r.choice([64, 128]))
        dtype = [torch.float16, torch.bfloat16][int(r.integers(2))]
        batch = int(r.integers(1, 40))
        ql = [int(n) for n in r.integers(0, int(r.choice([2, 5, 40, 300])), batch)]
        kl = [n + int(r.integers(0, 900)) for n in ql]
        q = normal(seed, sum(ql), heads, dim, dtype=dtype)
        k, v = (normal(seed + s, sum(kl), kv_heads, dim, dtype=dtype) for s in (1, 2))
        check_attention(q, k, v, ql, kl, causal=bool(r.integers(2)))


@gpu
@pytest.mark.parametrize("scale", [0.0, 1.0, 20.0, -0.3])
def test_attention_scales(scale):
    """Scores of several hundred (one key takes all), equal scores, a negative scale."""
    for ql, kl in (([200, 60], None), ([1, 2], [300, 1500])):
        tk = sum(ql if kl is None else kl)
        q, k, v = normal(1, sum(ql), 4, 64), normal(2, tk, 2, 64), normal(3, tk, 2, 64)
        check_attention(q, k, v, ql, kl, scale=scale)


@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_rising_and_falling_scores(dtype):
    """The largest score comes last, or first, by far: the running maximum moves in every tile or never again."""
    n, D = 700, 64
    for sign in (1.0, -1.0):
        ramp = torch.linspace(-1, 1, n, device="cuda").mul(sign)
        k = (ramp[:, None, None] * torch.ones(n, 1, D, device="cuda") * 4).to(dtype)
        q = torch.ones(n, 2, D, device="cuda", dtype=dtype)
        v = normal(5, n, 1, D, dtype=dtype)
        check_attention(q, k, v, [n], None)
        check_attention(q[:1], k, v, [1], [n])


@gpu
@pytest.mark.parametrize("heads,kv_heads,dim,ql,kl", [
    (16, 2, 64, [3, 0, 0], [2000, 5, 700]),  # as many queries as sequences, but one sequence has them all
    (32, 4, 128, [0, 5, 0, 0, 0], [10, 3000, 1, 1, 900]),
    (16, 2, 64, [0, 40] + [0] * 38, [900, 2600] + [7] * 38),
    (80, 1, 64, [1, 1], [300, 2000]),  # a group of more heads than the token tile's rows
    (40, 1, 256, [1, 1, 1], [1500, 7, 64]),
    (64, 1, 128, [1, 1], [1030, 2500]),
    (24, 3, 96, [2], [1400]),
    (12, 2, 128, [257, 1, 64], [2448, 1099, 64]),
])
def test_attention_uneven_batches(heads, kv_heads, dim, ql, kl):
    for causal in (True, False):
        q = normal(1, sum(ql), heads, dim)
        k, v = normal(2, sum(kl), kv_heads, dim), normal(3, sum(kl), kv_heads, dim)
        check_attention(q, k, v, ql, kl, causal)


@gpu
def test_attention_views():
    """Parts of one projection's output, heads before tokens, int64 offsets, rows wider than the heads."""
    ql = [37, 1, 140]
    T, H, Hk, D = sum(ql), 8, 2, 64
    qkv = normal(1, T, H + 2 * Hk, D)
    q, k, v = qkv.split((H, Hk, Hk), dim=1)
    want = check_attention(q, k, v, ql, None)
    swapped = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(check_attention(*swapped, ql, None), want)
    assert torch.equal(fk().packed_attention(q, k, v, offsets(ql, torch.int64)), want)
    wide = torch.full((T, H * D + 24), 7.0, dtype=torch.float16, device="cuda")
    out = wide[:, :H * D].unflatten(1, (H, D))
    assert fk().packed_attention(q, k, v, offsets(ql), out=out) is out
    assert torch.equal(out, want) and bool((wide[:, H * D:] == 7.0).all())
    one_key = normal(9, 1, 2, D).expand(T, 2, D)  # every token has the same key
    check_attention(q, one_key, v, ql, None)


@gpu
@pytest.mark.parametrize("q_lengths,k_lengths", [([20, 9], None), ([1, 1], [70, 9]), ([1, 40], [500, 90])])
def test_attention_rows_of_no_sequence(q_lengths, k_lengths):
    """Rows behind the last sequence and before the first: 0 in a new output, left as they were in a given one."""
    tq, lead, rest = sum(q_lengths), 3, 150
    tk = sum(k_lengths or q_lengths)
    q = normal(1, lead + tq + rest, 4, 64)
    k, v = normal(2, lead + tk + rest, 2, 64), normal(3, lead + tk + rest, 2, 64)
    qo = offsets(q_lengths) + lead
    ko = None if k_lengths is None else offsets(k_lengths) + lead
    got = fk().packed_attention(q, k, v, qo, ko)
    want, tol = attention_reference(q[lead:lead + tq], k[lead:lead + tk], v[lead:lead + tk], q_lengths,
                                    k_lengths or q_lengths, 64 ** -0.5, True)
    within(got[lead:lead + tq], want, tol)
    assert not got[:lead].any() and not got[lead + tq:].any()
    out = torch.full_like(q, 5.0)
    fk().packed_attention(q, k, v, qo, ko, out=out)
    assert torch.equal(out[lead:lead + tq], got[lead:lead + tq])
    assert bool((out[:lead] == 5.0).all()) and bool((out[lead + tq:] == 5.0).all())
    # no sequence at all
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    none = fk().packed_attention(q, k, v, zero, zero)
    assert not none.any()


@gpu
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 65504.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_hidden_values_have_no_effect(dtype, bad):
    """NaN, infinities and the largest values in keys and values that a query does not see."""
    H, Hk, D = 8, 2, 64
    for ql, kl in (([40, 90, 33], [40, 90, 33]), ([1, 1, 1], [100, 513, 64]), ([70, 1, 20], [300, 80, 1000])):
        tq, tk = sum(ql), sum(kl)
        q, k, v = normal(1, tq, H, D, dtype=dtype), normal(2, tk, Hk, D, dtype=dtype), normal(3, tk, Hk, D, dtype=dtype)
        clean = fk().packed_attention(q, k, v, offsets(ql), offsets(kl))
        # the middle sequence's keys and values, and those of the first sequence's last 10 tokens
        k2, v2 = k.clone(), v.clone()
        for t in (k2, v2):
            t[kl[0]:kl[0] + kl[1]] = bad
            t[kl[0] - 10:kl[0]] = bad
        got = fk().packed_attention(q, k2, v2, offsets(ql), offsets(kl))
        torch.cuda.synchronize()
        assert torch.equal(got[ql[0] + ql[1]:], clean[ql[0] + ql[1]:])
        early = max(ql[0] - 10, 0)
        assert torch.equal(got[:early], clean[:early])
        if math.isnan(bad):
            assert bool(torch.isnan(got[early:ql[0] + ql[1]]).all())
        # values alone, in single elements: the other elements of the row, and the rows before it, stay
        v3 = v.clone()
        v3[kl[0] - 3, :, 5] = bad
        got = fk().packed_attention(q, k, v3, offsets(ql), offsets(kl))
        torch.cuda.synchronize()
        same = torch.ones_like(got, dtype=torch.bool)
        same[max(ql[0] - 3, 0):ql[0], :, 5] = False
        assert torch.equal(got[same], clean[same])
        if not math.isfinite(bad):
            touched = got[~same].float()
            assert bool((torch.isnan(touched) if math.isnan(bad) else touched == bad).all())


@gpu
@pytest.mark.parametrize("dtype,value", [(torch.float16, 65504.0), (torch.float16, -65504.0), (torch.float16, 6e-8),
                                         (torch.bfloat16, 1e30), (torch.bfloat16, 0.3)])
def test_attention_of_constant_values(dtype, value):
    """Equal values come out as they are, the type's largest among them, and none where nothing is seen."""
    for ql, kl in (([200, 30], [200, 30]), ([1, 1], [700, 3]), ([5, 130], [2000, 1500]), ([9], [4])):
        q, k = normal(1, sum(ql), 6, 64, dtype=dtype), normal(2, sum(kl), 2, 64, dtype=dtype)
        v = torch.full_like(k, value)
        got = fk().packed_attention(q, k, v, offsets(ql), offsets(kl))
        want = torch.full_like(got, value)
        if ql == [9]:
            want[:5] = 0.0
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@gpu
def test_attention_of_no_queries_or_keys():
    q, k, v = normal(1, 6, 4, 64), normal(2, 9, 2, 64), normal(3, 9, 2, 64)
    kernels = fk()
    assert not kernels.packed_attention(q, k[:0], v[:0], offsets([2, 4]), offsets([0, 0])).any()
    assert not kernels.packed_attention(q[:2], k[:0], v[:0], offsets([1, 1]), offsets([0, 0])).any()
    assert kernels.packed_attention(q[:0], k, v, offsets([0]), offsets([9])).shape == (0, 4, 64)
    assert kernels.packed_attention(q[:0], k[:0], v[:0], offsets([])).shape == (0, 4, 64)


@gpu
def test_attention_rows_do_not_depend_on_their_neighbours():
    """A sequence's rows have the same bits alone and in a batch of its kind, twice over."""
    ql = [65, 200, 129]
    q, k, v = normal(1, sum(ql), 8, 64), normal(2, sum(ql), 2, 64), normal(3, sum(ql), 2, 64)
    whole = fk().packed_attention(q, k, v, offsets(ql))
    assert torch.equal(fk().packed_attention(q, k, v, offsets(ql)), whole)


@gpu
def test_attention_offsets_are_held_to_the_tensors():
    """Offsets outside the tensors are held to them."""
    q, k, v = normal(1, 50, 4, 64), normal(2, 50, 2, 64), normal(3, 50, 2, 64)
    want = fk().packed_attention(q, k, v, offsets([20, 30]))
    far = torch.tensor([-5, 20, 70], dtype=torch.int32, device="cuda")
    assert torch.equal(fk().packed_attention(q, k, v, far), want)
    one = fk().packed_attention(q[:1], k, v, offsets([1]), torch.tensor([-9, 1 << 30], dtype=torch.int32, device="cuda"))
    ref, tol = attention_reference(q[:1], k, v, [1], [50], 64 ** -0.5, True)
    within(one, ref, tol)


@gpu
@pytest.mark.parametrize("nq", [1, 200])
def test_attention_far_offsets(nq):
    """Key rows beyond 2^32 elements from their tensor's start."""
    T, stride, D = (1 << 18) + 77, 1 << 14, 64
    buf = torch.empty((T, stride), dtype=torch.float16, device="cuda")
    k, v = buf[:, :D].unflatten(1, (1, D)), buf[:, D:2 * D].unflatten(1, (1, D))
    tail = 3000
    k[T - tail:] = normal(1, tail, 1, D)
    v[T - tail:] = normal(2, tail, 1, D)
    q = normal(3, nq, 4, D)
    ko = torch.tensor([T - tail, T], dtype=torch.int32, device="cuda")
    got = fk().packed_attention(q, k, v, offsets([nq]), ko)
    want, tol = attention_reference(q, k[T - tail:], v[T - tail:], [nq], [tail], D ** -0.5, True)
    within(got, want, tol)


@gpu
def test_attention_long_keys():
    """One token against 70,000 keys, sequences of very unequal length, chunks that end everywhere."""
    for kl in ([70000], [9, 40000, 700], [513, 511, 1024, 1025, 1, 0, 1537, 512, 2047, 3], [600] * 40,
               [2000 + 37 * i for i in range(24)]):
        ql = [1] * len(kl)
        q = normal(1, len(kl), 8, 128, dtype=torch.bfloat16)
        k, v = (normal(s, sum(kl), 1, 128, dtype=torch.bfloat16) for s in (2, 3))
        check_attention(q, k, v, ql, kl)


@gpu
@pytest.mark.parametrize("batch", [63, 64, 65, 127, 300, 4095, 4096, 4097, 9000])
def test_attention_many_sequences(batch):
    """Short sequences by the hundreds and thousands, some empty: prompts, single tokens, tokens with long keys."""
    r = np.random.default_rng(batch)
    ql = [int(n) for n in r.integers(0, 4, batch)]
    q, k, v = normal(1, sum(ql), 2, 32), normal(2, sum(ql), 1, 32), normal(3, sum(ql), 1, 32)
    seqs = np.repeat(np.arange(batch), ql)
    starts = np.concatenate([[0], np.cumsum(ql)])

    def check(got, seq_of, k_starts, k_len, pos):
        """Every row against its own sequence's keys, padded to the longest."""
        top = int(k_len.max())
        cols = torch.arange(top, device="cuda")
        first = torch.from_numpy(k_starts[seq_of]).cuda()
        idx = (first[:, None] + cols).clamp(max=k2.shape[0] - 1)
        kk, vv = k2[idx, 0].double(), v2[idx, 0].double()  # [rows, top, D]
        seen = torch.from_numpy(pos).cuda()[:, None] >= cols
        for h in range(q2.shape[1]):
            qq = q2[:, h].double()
            s = (kk * qq[:, None]).sum(-1) * 32 ** -0.5
            p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
            want = (p[..., None] * vv).sum(1)
            av = (p[..., None] * vv.abs()).sum(1)
            d = 40 * E * ((kk * qq[:, None]).abs().sum(-1) * 32 ** -0.5).amax(-1, keepdim=True)
            tol = (2.0 ** -10 * want.abs() + TINY[q.dtype] + av * (2.0 ** -11 + 2 * d + 2.0 ** -20 + top * E)
                   + 2.0 ** -25 * ((vv.abs() * seen[..., None]).sum(1) + seen.sum(-1, keepdim=True) * want.abs()))
            within(got[:, h], want, tol, f"{batch} sequences")

    q2, k2, v2 = q, k, v
    check(fk().packed_attention(q, k, v, offsets(ql)), seqs, starts, np.asarray(ql),
          np.arange(len(seqs)) - starts[seqs])
    kl = r.integers(1, 9, batch)
    q2, k2, v2 = normal(4, batch, 2, 32), normal(5, int(kl.sum()), 1, 32), normal(6, int(kl.sum()), 1, 32)
    check(fk().packed_attention(q2, k2, v2, offsets([1] * batch), offsets(kl)), np.arange(batch),
          np.concatenate([[0], np.cumsum(kl)]), kl, kl - 1)


@gpu
@pytest.mark.parametrize("q_cap,lengths", [(64, ([40, 24], [10, 30, 24])), (2, ([1, 1], [1, 1]))])
def test_attention_in_a_graph(q_cap, lengths):
    """Captured once, replayed with other offsets and inputs, two graphs in turn, against eager calls."""
    H, Hk, D, Tk = 8, 2, 64, 3000
    bufs = [(normal(i, q_cap, H, D), normal(i + 5, Tk, Hk, D), normal(i + 9, Tk, Hk, D)) for i in range(2)]
    qo = torch.tensor([0, q_cap // 2, q_cap], dtype=torch.int32, device="cuda")
    ko = torch.tensor([0, 1000, Tk], dtype=torch.int32, device="cuda")
    kernels = fk()
    kernels.packed_attention(*bufs[0], qo, ko)
    graphs, outs = [], []
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kernels.packed_attention(*b, qo, ko))
        graphs.append(g)
    for step, cut in enumerate((0, 777, 2999, 100)):
        ko[1] = cut
        for b in bufs:
            b[0].copy_(normal(100 + step, q_cap, H, D))
        eager = [kernels.packed_attention(*b, qo, ko) for b in bufs]
        for o in outs:
            o.fill_(math.nan)
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert torch.equal(o, e)


@gpu
def test_attention_on_two_streams():
    q, k, v = normal(1, 4, 8, 128), normal(2, 20000, 2, 128), normal(3, 20000, 2, 128)
    qo, ko = offsets([1, 1, 1, 1]), offsets([5000] * 4)
    q2 = normal(7, 4, 8, 128)
    kernels = fk()
    want = [kernels.packed_attention(x, k, v, qo, ko) for x in (q, q2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, x in zip(streams, (q, q2)):
            with torch.cuda.stream(s):
                got.append(kernels.packed_attention(x, k, v, qo, ko))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
def test_attention_without_a_workspace():
    """A C caller that gives no workspace gets the rows without a split: the same within the tolerance."""
    from gliner_decide.device import stream_handle
    H, Hk, D, nk = 8, 2, 128, 9000
    q, k, v = normal(1, 1, H, D), normal(2, nk, Hk, D), normal(3, nk, Hk, D)
    out = torch.empty_like(q)
    qo, ko = offsets([1]), offsets([nk])
    st = N.lib().gd_packed_attention(N.GdTokens(q.data_ptr(), 0, D), N.GdTokens(k.data_ptr(), Hk * D, D),
                                     N.GdTokens(v.data_ptr(), Hk * D, D), qo.data_ptr(), ko.data_ptr(), 1, 1, nk, H, Hk,
                                     D, N.GD_F16, D ** -0.5, N.GD_PACKED_CAUSAL, out.data_ptr(), H * D, None, 0,
                                     stream_handle())
    assert st == N.GD_OK
    want, tol = attention_reference(q, k, v, [1], [nk], D ** -0.5, True)
    within(out, want, tol)


def _attention_status(q=(FAKE, 512, 64), k=(2 * FAKE, 128, 64), v=(3 * FAKE, 128, 64), qo=4 * FAKE, ko=5 * FAKE, batch=2,
                      tq=10, tk=20, heads=8, kv_heads=2, dim=64, dtype=N.GD_F16, scale=0.125, flags=1, out=6 * FAKE,
                      ldo=512, work=None, size=0):
    return N.lib().gd_packed_attention(N.GdTokens(*q), N.GdTokens(*k), N.GdTokens(*v), qo, ko, batch, tq, tk, heads,
                                       kv_heads, dim, dtype, scale, flags, out, ldo, work, size, None)


@pytest.mark.parametrize("status,kwargs", [
    (N.GD_ERR_INVALID_ARGUMENT, dict(dtype=N.GD_F32)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(flags=4)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(scale=math.nan)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(scale=math.inf)),
    (N.GD_ERR_SHAPE, dict(batch=-1)),
    (N.GD_ERR_SHAPE, dict(tq=1 << 31)),
    (N.GD_ERR_SHAPE, dict(tk=-1)),
    (N.GD_ERR_SHAPE, dict(heads=7)),
    (N.GD_ERR_SHAPE, dict(kv_heads=0)),
    (N.GD_ERR_SHAPE, dict(dim=80)),
    (N.GD_ERR_SHAPE, dict(ko=None)),  # 20 keys of 10 tokens
    (N.GD_ERR_SHAPE, dict(ldo=504)),
    (N.GD_ERR_SHAPE, dict(ldo=516)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(q=(FAKE + 2, 512, 64))),
    (N.GD_ERR_INVALID_ARGUMENT, dict(k=(2 * FAKE, 132, 64))),
    (N.GD_ERR_INVALID_ARGUMENT, dict(v=(3 * FAKE, 128, 60))),
    (N.GD_ERR_SHAPE, dict(v=(3 * FAKE, -128, 64))),
    (N.GD_ERR_INVALID_ARGUMENT, dict(q=(None, 512, 64))),
    (N.GD_ERR_INVALID_ARGUMENT, dict(k=(None, 128, 64))),
    (N.GD_ERR_INVALID_ARGUMENT, dict(qo=None)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(out=None)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(out=6 * FAKE + 8)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(out=FAKE)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(out=3 * FAKE + 19 * 256)),  # v's last row
    (N.GD_ERR_INVALID_ARGUMENT, dict(work=FAKE + 4, size=64)),
])
def test_attention_refusals(status, kwargs):
    assert _attention_status(**kwargs) == status
    assert N.last_error()


@pytest.mark.parametrize("batch", [1, 16, 4096, 1 << 20])
def test_attention_workspace_does_not_grow_with_the_batch(batch):
    """Single tokens over 2^28 keys in all: parts for the chunks, not for every sequence."""
    size = N.lib().gd_packed_attention_workspace(batch, batch, 1 << 28, 32, 8, 128)
    assert 0 < size <= 64 << 20


def test_attention_of_nothing_without_device():
    assert _attention_status(tq=0, q=(None, 0, 64), out=None) == N.GD_OK
    assert N.lib().gd_packed_attention_workspace(0, 5, 5, 8, 2, 64) == 0
    assert N.lib().gd_packed_attention_workspace(1, 5, 5, 7, 2, 64) == 0


# ---------------------------------------------------------------------------
# projection
# ---------------------------------------------------------------------------
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def activate(y, kind):
    if kind == "relu":
        return torch.where(y > 0, y, torch.where(y <= 0, 0.0, y))
    if kind == "gelu":
        return 0.5 * y * torch.special.erfc(-y / math.sqrt(2.0))
    if kind == "gelu_tanh":
        return y * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
    if kind == "silu":
        return y * torch.special.expit(y)
    return y


def projection_reference(x, w, bias, residual, kind, scale):
    K = x.shape[-1]
    xx, ww = x.double().reshape(-1, K), w.double()
    acc = xx @ ww.T.contiguous()
    mag = xx.abs() @ ww.abs().T.contiguous()
    b = torch.zeros(w.shape[0], dtype=torch.float64, device=x.device) if bias is None else bias.double()
    y = activate(acc + b, kind)
    slope = 1.0 if kind in ("none", "relu") else 1.13
    tol = slope * (K + 8) * E * (mag + b.abs()) + 2.0 ** -15 * y.abs() * (kind not in ("none", "relu"))
    out = scale * y
    tol = abs(scale) * tol + 4 * E * out.abs()
    if residual is not None:
        r = residual.double().reshape(out.shape)
        tol = tol + 4 * E * r.abs()
        out = out + r
    tol = tol + HALF_STEP[x.dtype] * (out.abs() + tol) + TINY[x.dtype]
    shape = x.shape[:-1] + (w.shape[0],)
    return out.reshape(shape), tol.reshape(shape)


def check_projection(x, w, bias=None, residual=None, activation="none", scale=1.0, **kw):
    want, tol = projection_reference(x, w, bias, residual, activation, scale)
    got = fk().projection(x, w, bias, residual, activation=activation, scale=scale, **kw)
    assert got.shape == want.shape and got.dtype == x.dtype
    within(got, want, tol, f"projection {tuple(x.shape)} x {tuple(w.shape)}")
    return got


SIZES = [(1, 1, 1), (1, 4096, 1024), (1, 1000, 4096), (2, 130, 72), (3, 7, 5), (4, 64, 1024), (5, 129, 1000),
         (8, 1024, 4096), (16, 256, 264), (17, 2048, 64), (31, 100, 8), (33, 384, 520), (64, 1024, 512), (65, 65, 65),
         (100, 1000, 1016), (128, 128, 64), (130, 257, 136), (257, 512, 1024), (300, 1001, 333), (777, 1000, 1024),
         (1030, 640, 96), (2500, 1024, 256)]


@gpu
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_projection_sizes(dtype, activation):
    for i, (m, n, k) in enumerate(SIZES):
        x = normal(3 * i, m, k, dtype=dtype)
        w = normal(3 * i + 1, n, k, dtype=dtype, scale=2.0 * k ** -0.5)
        b = normal(3 * i + 2, n, dtype=dtype) if i % 3 else None
        r = normal(3 * i + 3, m, n, dtype=dtype) if i % 2 else None
        check_projection(x, w, b, r, activation, 1.0 if i % 5 else 0.25)


@gpu
@pytest.mark.parametrize("seed", range(10))
def test_projection_drawn_sizes(seed):
    r = np.random.default_rng(100 + seed)
    for _ in range(6):
        m, n, k = (int(np.exp(r.uniform(0, np.log(hi)))) for hi in (3000, 3000, 2500))
        if r.random() < 0.5:
            k = -(-k // 8) * 8
        dtype = [torch.float16, torch.bfloat16][int(r.integers(2))]
        check_projection(normal(seed, m, k, dtype=dtype), normal(seed + 1, n, k, dtype=dtype, scale=k ** -0.5),
                         normal(seed + 2, n, dtype=dtype) if r.random() < 0.5 else None,
                         normal(seed + 3, m, n, dtype=dtype) if r.random() < 0.5 else None,
                         ACTIVATIONS[int(r.integers(5))], float(r.choice([1.0, -0.5, 0.0])))


@gpu
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("m", [1, 40, 300])
def test_projection_activation_range(activation, m):
    """The whole range of an activation's argument: x of one column, weight 1, so y is x itself."""
    for dtype in (torch.float16, torch.bfloat16):
        n = 1500
        w = torch.linspace(-12, 12, n, device="cuda")[:, None].to(dtype)
        x = torch.ones((m, 1), device="cuda", dtype=dtype)
        check_projection(x, w, None, None, activation)
        big = torch.tensor([[3e4], [-3e4], [90.0], [-90.0], [0.0], [-0.0], [1e-4], [-1e-4]], device="cuda", dtype=dtype)
        check_projection(x, big, None, None, activation)
        special = torch.tensor([[math.inf], [math.nan]], device="cuda", dtype=dtype)
        got = fk().projection(x, special, activation=activation)
        assert bool(torch.isinf(got[:, 0]).all()) and bool(torch.isnan(got[:, 1]).all())


@gpu
@pytest.mark.parametrize("m", [1, 6, 50, 400])
def test_projection_views_and_outputs(m):
    """Rows at other strides, unaligned starts, leading axes, a given output inside a larger one, the residual itself."""
    n, k = 200, 136
    buf = normal(1, m + 2, k + 40)
    wbuf = normal(2, n, k + 9, scale=0.1)
    b = normal(3, n)
    r = normal(4, m, n)
    for x in (buf[:m, :k], buf[1:m + 1, 8:8 + k], buf[:m, 3:3 + k], buf[:m, 0:2 * (k // 2):1][:, :k]):
        for w in (wbuf[:, :k], wbuf[:, 5:5 + k]):
            want = check_projection(x, w, b, r, "gelu", 0.5)
            dense = check_projection(x.contiguous(), w.contiguous(), b, r, "gelu", 0.5)
            assert want.shape == dense.shape
    x, w = buf[:m, :k], wbuf[:, :k].contiguous()
    want = check_projection(x, w, b, r)
    assert torch.equal(check_projection(x.t().contiguous().t(), w, b, r), fk().projection(x.contiguous(), w, b, r))
    hold = torch.full((m + 2, n + 13), 9.0, dtype=torch.float16, device="cuda")
    out = hold[1:m + 1, 5:5 + n]
    assert fk().projection(x, w, b, r, out=out) is out
    assert torch.equal(out, want)
    hold[1:m + 1, 5:5 + n] = 9.0
    assert bool((hold == 9.0).all())
    inplace = r.clone()
    fk().projection(x, w, b, inplace, out=inplace)
    assert torch.equal(inplace, want)
    lead = check_projection(x.reshape(1, m, 1, k), w, b, r.reshape(1, m, 1, n))
    assert torch.equal(lead.reshape(m, n), want)
    rows = x[:1].expand(m, k)
    check_projection(rows, w, b, r)


@gpu
def test_projection_rows_apart():
    """NaN and infinities in a row of x stay in that row, those of a row of w in that column; no rows, no columns."""
    for m, n, k in ((5, 70, 64), (40, 200, 136), (300, 260, 72)):
        x, w = normal(1, m, k), normal(2, n, k, scale=0.1)
        clean = fk().projection(x, w)
        x2, w2 = x.clone(), w.clone()
        x2[m - 1, 3], w2[n - 1, 5] = math.nan, math.inf
        got = fk().projection(x2, w2)
        torch.cuda.synchronize()
        assert torch.equal(got[:-1, :-1], clean[:-1, :-1])
        assert bool(torch.isnan(got[-1]).all()) and not bool(torch.isfinite(got[:, -1]).any())
    assert fk().projection(x[:0], w).shape == (0, n)
    assert fk().projection(x, w[:0]).shape == (m, 0)


@gpu
@pytest.mark.parametrize("m", [1, 30, 500])
def test_projection_in_a_graph(m):
    x, w, r = normal(1, m, 520), normal(2, 300, 520, scale=0.1), normal(3, m, 300)
    kernels = fk()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = kernels.projection(x, w, None, r, activation="silu")
    for step in range(4):
        x.copy_(normal(50 + step, m, 520))
        eager = kernels.projection(x, w, None, r, activation="silu")
        out.fill_(math.nan)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@gpu
def test_projection_far_rows():
    """Rows of x, the residual and the output beyond 2^32 elements from their start."""
    stride, m, n, k = 1 << 22, 1030, 256, 128
    buf = torch.empty((m, stride), dtype=torch.float16, device="cuda")
    x, r, out = buf[:, :k], buf[:, 4096:4096 + n], buf[:, 8192:8192 + n]
    x.copy_(normal(1, m, k))
    r.copy_(normal(2, m, n))
    w = normal(3, n, k, scale=0.1)
    other = torch.empty((m, stride), dtype=torch.float16, device="cuda")[:, :n]
    want, tol = projection_reference(x, w, None, r, "none", 1.0)
    fk().projection(x, w, None, r, out=other)
    within(other, want, tol)
    # few rows, and a weight of far rows
    wfar = buf[:, 20000:20000 + k]
    wfar.copy_(normal(4, m, k, scale=0.1))
    check_projection(normal(5, 3, k), wfar)
    check_projection(normal(6, 300, k), wfar)


def _projection_status(x=(FAKE, 64), w=(2 * FAKE, 64), bias=3 * FAKE, residual=(4 * FAKE, 128), out=5 * FAKE, ldo=128,
                       m=8, n=128, k=64, act=0, scale=1.0, dtype=N.GD_F16):
    return N.lib().gd_projection(N.GdRows(*x), N.GdRows(*w), bias, N.GdRows(*residual), out, ldo, m, n, k, act, scale,
                                 dtype, None)


@pytest.mark.parametrize("status,kwargs", [
    (N.GD_ERR_INVALID_ARGUMENT, dict(dtype=N.GD_F32)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(act=5)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(act=-1)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(scale=math.inf)),
    (N.GD_ERR_SHAPE, dict(m=-1)),
    (N.GD_ERR_SHAPE, dict(k=0)),
    (N.GD_ERR_SHAPE, dict(n=1 << 31)),
    (N.GD_ERR_SHAPE, dict(x=(FAKE, 63))),
    (N.GD_ERR_SHAPE, dict(w=(2 * FAKE, 0))),
    (N.GD_ERR_SHAPE, dict(ldo=127)),
    (N.GD_ERR_SHAPE, dict(residual=(4 * FAKE, 100))),
    (N.GD_ERR_INVALID_ARGUMENT, dict(x=(None, 64))),
    (N.GD_ERR_INVALID_ARGUMENT, dict(w=(None, 64))),
    (N.GD_ERR_INVALID_ARGUMENT, dict(out=None)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(x=(FAKE + 1, 64))),
    (N.GD_ERR_INVALID_ARGUMENT, dict(out=FAKE)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(out=2 * FAKE + 64)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(out=3 * FAKE)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(out=4 * FAKE, ldo=136)),  # the residual at another stride
    (N.GD_ERR_INVALID_ARGUMENT, dict(out=4 * FAKE + 2)),
])
def test_projection_refusals(status, kwargs):
    assert _projection_status(**kwargs) == status
    assert N.last_error()


# ---------------------------------------------------------------------------
# block_norm
# ---------------------------------------------------------------------------
NORM_ERR = 2.0 ** -18


def norm_reference(x, dx, w, b, eps, layer):
    """(norm, tolerance) of rows x that are off by at most dx."""
    centre = x.mean(-1, keepdim=True) if layer else torch.zeros_like(x[..., :1])
    rs = 1.0 / torch.sqrt(((x - centre) ** 2).mean(-1, keepdim=True) + eps)
    z = (x - centre) * rs
    # x moves by dx, its mean and spread by no more than the row's largest dx; the arithmetic by NORM_ERR of the
    # row's largest entry before the mean is taken off
    top = x.abs().amax(-1, keepdim=True) * rs
    move = dx.amax(-1, keepdim=True) * rs
    tol = (NORM_ERR * (top + z.abs() * (1.0 + top)) + 2 * move + z.abs() * move * 2) * w.abs()
    out = z * w
    if b is not None:
        out = out + b
    return out, tol + 4 * E * out.abs()


def block_norm_reference(y, res, post, pre, gate, scale, eps, layer):
    """post, pre: (weight, bias) or None.  (h, tol, n, tol)."""
    def wide(t):
        return None if t is None else t.double()
    z = y.double()
    dz = torch.zeros_like(z)
    if post is not None:
        z, dz = norm_reference(z, dz, wide(post[0]), wide(post[1]), eps, layer)
    if gate is not None:
        g = gate.double()
        z, dz = z * g, dz * g.abs() + 2 * E * (z * g).abs()
    r = res.double()
    h = r + scale * z
    dh = abs(scale) * dz + 4 * E * (r.abs() + (scale * z).abs())
    n, dn = norm_reference(h, dh, wide(pre[0]), wide(pre[1]), eps, layer)
    return (h, dh + HALF_STEP[res.dtype] * (h.abs() + dh) + TINY[res.dtype], n,
            dn + HALF_STEP[y.dtype] * (n.abs() + dn) + TINY[y.dtype])


def check_block_norm(y, res, pre, post=None, gate=None, scale=1.0, eps=1e-6, kind="rms", out=None):
    hw, ht, nw, nt = block_norm_reference(y, res, post, pre, gate, scale, eps, kind == "layer")
    h, n = fk().block_norm(y, res, pre_weight=pre[0], pre_bias=pre[1], post_weight=None if post is None else post[0],
                           post_bias=None if post is None else post[1], gate=gate, scale=scale, eps=eps, kind=kind,
                           out=out)
    assert h.dtype == res.dtype and n.dtype == y.dtype and h.shape == res.shape and n.shape == y.shape
    within(h, hw, ht, f"h {tuple(y.shape)}")
    within(n, nw, nt, f"n {tuple(y.shape)}")
    return h, n


@gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("stream", ["same", "fp32"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_block_norm_sizes(dtype, stream, kind):
    sd = torch.float32 if stream == "fp32" else dtype
    sizes = [(1, 1), (3, 2), (2, 7), (5, 64), (300, 72), (9, 255), (4, 256), (33, 512), (7, 520), (5, 1000), (1, 1024),
             (130, 1024), (6, 1025), (2, 2047), (17, 2048), (5, 4096), (3, 4104), (2, 5001), (3, 8192), (2, 16384),
             (1, 32767), (2, 32768)]
    for i, (rows, cols) in enumerate(sizes):
        y, res = normal(i, rows, cols, dtype=dtype), normal(i + 1, rows, cols, dtype=sd)
        w = [normal(i + 2 + j, cols, dtype=dtype, mean=1.0, scale=0.2) for j in range(2)]
        b = [normal(i + 5 + j, cols, dtype=dtype, scale=0.2) if (i + j) % 3 else None for j in range(2)]
        gate = (None, normal(i + 9, cols, dtype=dtype), normal(i + 9, rows, cols, dtype=dtype))[i % 3]
        check_block_norm(y, res, (w[0], b[0]), (w[1], b[1]) if i % 4 else None, gate, (1.0, 0.3)[i % 2], kind=kind)


@gpu
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_block_norm_rows_of_all_kinds(kind):
    """Zero, constant, tiny, huge, off-centre and one-entry rows."""
    C_ = 1000
    rows = torch.zeros(8, C_, device="cuda")
    rows[1] = 3.0
    rows[2] = 1e-4 * normal(1, C_).float()
    rows[3] = 6e4 * torch.sign(normal(2, C_).float())
    rows[4] = 500.0 + normal(3, C_).float()
    rows[5, 17] = 1e3
    rows[6] = -2.0
    rows[7] = normal(4, C_).float()
    w, b = normal(5, C_, mean=1.0, scale=0.2), normal(6, C_, scale=0.2)
    for eps in (1e-7, 1e-3):
        zero = torch.zeros(8, C_, dtype=torch.float16, device="cuda")
        check_block_norm(rows.half(), zero, (w, b), (w, b), kind=kind, eps=eps)
        check_block_norm(zero, rows.half(), (w, b), None, kind=kind, eps=eps)
        check_block_norm(rows.half(), rows.float(), (w, b), None, None, 0.0, kind=kind, eps=eps)


@gpu
@pytest.mark.parametrize("cols", [64, 136, 1000, 1024, 4096, 999])
def test_block_norm_gates_views_and_outputs(cols):
    B, L = 3, 11
    y, res = normal(1, B, L, cols), normal(2, B, L, cols)
    w, b = normal(3, cols, mean=1.0, scale=0.2), normal(4, cols, scale=0.2)
    for shape in ((cols,), (1, 1, cols), (B, 1, cols), (1, L, cols), (L, cols), (B, L, cols)):
        check_block_norm(y, res, (w, None), (w, b), normal(5, *shape), 0.5)
    gate = normal(5, B, 1, cols).expand(B, L, cols)
    want = check_block_norm(y, res, (w, b), (w, b), gate, kind="layer")
    # rows of a wider tensor, unaligned columns, given outputs inside larger ones
    yy = normal(7, B * L, cols + 21)
    yy[:, 5:5 + cols] = y.reshape(-1, cols)
    rr = normal(8, B * L, cols + 16)
    rr[:, 8:8 + cols] = res.reshape(-1, cols)
    hh = torch.full((B * L + 1, cols + 8), 4.0, dtype=torch.float16, device="cuda")
    nn = torch.full((B * L + 1, cols + 3), 4.0, dtype=torch.float16, device="cuda")
    out = (hh[:-1, 8:8 + cols], nn[:-1, 1:1 + cols])
    got = check_block_norm(yy[:, 5:5 + cols], rr[:, 8:8 + cols], (w, b), (w, b), gate.reshape(-1, cols), kind="layer",
                           out=out)
    assert got[0] is out[0] and got[1] is out[1]
    ht = block_norm_reference(y, res, (w, b), (w, b), gate, 1.0, 1e-6, True)
    within(got[0], want[0].double().reshape(-1, cols), 2 * ht[1].reshape(-1, cols))
    for t, lo in ((hh, 8), (nn, 1)):
        t[:-1, lo:lo + cols] = 4.0
        assert bool((t == 4.0).all())
    # in place: h the residual, n the block's output; and the other way round
    for swap in (False, True):
        y2, r2 = y.clone(), res.clone()
        o = (y2, r2) if swap else (r2, y2)
        fk().block_norm(y2, r2, pre_weight=w, pre_bias=b, post_weight=w, post_bias=b, gate=gate, kind="layer", out=o)
        assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])
    # a residual in fp32, in place
    r32 = res.float()
    check_block_norm(y, r32.clone(), (w, b), (w, b), gate, kind="layer")
    got = fk().block_norm(y, r32, pre_weight=w, out=(r32, torch.empty_like(y)))
    assert got[0] is r32
    assert fk().block_norm(y[:0], res[:0], pre_weight=w)[0].shape == (0, L, cols)


@gpu
def test_block_norm_rows_apart():
    for cols in (64, 1024, 5000, 777):
        y, res = normal(1, 40, cols), normal(2, 40, cols)
        w = normal(3, cols)
        clean = fk().block_norm(y, res, pre_weight=w, post_weight=w)
        y[17, 3], res[21, 5] = math.nan, math.inf
        got = fk().block_norm(y, res, pre_weight=w, post_weight=w)
        keep = [i for i in range(40) if i not in (17, 21)]
        for g, c in zip(got, clean):
            assert torch.equal(g[keep], c[keep])
        assert bool(torch.isnan(got[1][17]).all())


@gpu
def test_block_norm_in_a_graph_and_far_rows():
    y, res, w = normal(1, 50, 1024), normal(2, 50, 1024), normal(3, 1024)
    kernels = fk()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = kernels.block_norm(y, res, pre_weight=w, post_weight=w)
    for step in range(4):
        y.copy_(normal(10 + step, 50, 1024))
        eager = kernels.block_norm(y, res, pre_weight=w, post_weight=w)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])
    stride, rows = 1 << 22, 1030
    buf = torch.empty((rows, stride), dtype=torch.float16, device="cuda")
    far = [buf[:, 2048 * i:2048 * i + 1024] for i in range(3)]
    for i, t in enumerate(far):
        t.copy_(normal(20 + i, rows, 1024))
    other = torch.empty((rows, stride), dtype=torch.float16, device="cuda")
    check_block_norm(far[0], far[1], (w, None), (w, None), far[2], out=(other[:, :1024], other[:, 4096:5120]))


def _norm_status(y=(FAKE, 64), res=(2 * FAKE, 64), gate=(None, 0), per=1, post_w=3 * FAKE, post_b=None, pre_w=4 * FAKE,
                 pre_b=None, h=5 * FAKE, ldh=64, n=6 * FAKE, ldn=64, rows=8, cols=64, eps=1e-6, scale=1.0, kind=0,
                 dtype=N.GD_F16, stream_dtype=N.GD_F16):
    return N.lib().gd_block_norm(N.GdRows(*y), N.GdRows(*res), N.GdRows(*gate), per, post_w, post_b, pre_w, pre_b, h, ldh,
                                 n, ldn, rows, cols, eps, scale, kind, dtype, stream_dtype, None)


@pytest.mark.parametrize("status,kwargs", [
    (N.GD_ERR_INVALID_ARGUMENT, dict(dtype=N.GD_F32)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(stream_dtype=N.GD_BF16)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(kind=2)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(eps=0.0)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(eps=math.nan)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(scale=math.nan)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(post_w=None, post_b=FAKE)),
    (N.GD_ERR_SHAPE, dict(rows=-1)),
    (N.GD_ERR_SHAPE, dict(cols=0)),
    (N.GD_ERR_SHAPE, dict(cols=32769)),
    (N.GD_ERR_SHAPE, dict(gate=(7 * FAKE, 64), per=0)),
    (N.GD_ERR_SHAPE, dict(gate=(7 * FAKE, 60), per=2)),
    (N.GD_ERR_SHAPE, dict(y=(FAKE, 63))),
    (N.GD_ERR_SHAPE, dict(ldn=60)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(y=(None, 64))),
    (N.GD_ERR_INVALID_ARGUMENT, dict(pre_w=None)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(h=None)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(n=6 * FAKE + 1)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(stream_dtype=N.GD_F32, h=5 * FAKE + 2)),
    (N.GD_ERR_INVALID_ARGUMENT, dict(h=6 * FAKE + 128)),  # over n
    (N.GD_ERR_INVALID_ARGUMENT, dict(h=FAKE + 128)),  # over y, shifted
    (N.GD_ERR_INVALID_ARGUMENT, dict(h=2 * FAKE, ldh=72)),  # the residual at another stride
    (N.GD_ERR_INVALID_ARGUMENT, dict(stream_dtype=N.GD_F32, h=FAKE)),  # y as fp32
    (N.GD_ERR_INVALID_ARGUMENT, dict(n=3 * FAKE)),  # a weight
    (N.GD_ERR_INVALID_ARGUMENT, dict(gate=(7 * FAKE, 64), h=7 * FAKE + 64)),
])
def test_block_norm_refusals(status, kwargs):
    assert _norm_status(**kwargs) == status
    assert N.last_error()


@pytest.mark.parametrize("shift,apart", [(64, True), (63, False), (4096 - 64, True), (4096 - 63, False),
                                         (4096 * 3 + 100, True), (4096 * 3 + 20, False), (0, False)])
def test_outputs_between_an_inputs_columns(shift, apart):
    """n between the columns of the gate's rows is refused only where they touch (the call is refused in any case,
    for an h shifted over y)."""
    st = _norm_status(gate=(FAKE, 4096), n=FAKE + 2 * shift, ldn=4096, y=(1 << 30, 64), h=(1 << 30) + 128)
    assert st == N.GD_ERR_INVALID_ARGUMENT
    assert ("gate" not in N.last_error()) == apart, N.last_error()


@gpu
def test_python_refusals():
    k = fk()
    q, kv = normal(1, 10, 4, 64), normal(2, 10, 2, 64)
    qo = offsets([10])
    with pytest.raises(ValueError):
        k.packed_attention(q.cpu(), kv, kv, qo)
    with pytest.raises(ValueError):
        k.packed_attention(q, kv.cpu(), kv, qo)
    with pytest.raises(ValueError):
        k.packed_attention(q, kv, kv, qo.cpu())
    with pytest.raises(TypeError):
        k.packed_attention(q.float(), kv, kv, qo)
    with pytest.raises(TypeError):
        k.packed_attention(q, kv.bfloat16(), kv, qo)
    for bad in (dict(q=q[0]), dict(k=kv[:5]), dict(k=kv[..., :32], v=kv[..., :32]), dict(q_offsets=qo[None]),
                dict(k_offsets=offsets([5, 5])), dict(out=normal(1, 9, 4, 64)), dict(q=q.transpose(1, 2)),
                dict(k=kv[:5], v=kv[:5])):
        with pytest.raises(N.GlinerDecideError):
            k.packed_attention(**{**dict(q=q, k=kv, v=kv, q_offsets=qo), **bad})
    x, w = normal(1, 6, 64), normal(2, 32, 64)
    with pytest.raises(TypeError):
        k.projection(x, w.bfloat16())
    for bad in (dict(weight=w[:, :60]), dict(activation="tanh"), dict(bias=normal(1, 31)), dict(residual=normal(1, 6, 31)),
                dict(out=normal(1, 5, 32)), dict(weight=w[0])):
        with pytest.raises(N.GlinerDecideError):
            k.projection(**{**dict(x=x, weight=w), **bad})
    y, r, p = normal(1, 6, 64), normal(2, 6, 64), normal(3, 64)
    with pytest.raises(TypeError):
        k.block_norm(y, r.bfloat16(), pre_weight=p)
    for bad in (dict(residual=r[:5]), dict(kind="group"), dict(pre_weight=None), dict(gate=normal(1, 5, 64)),
                dict(gate=normal(1, 32)), dict(gate=normal(1, 1, 6, 64)), dict(pre_bias=p[:5]), dict(post_bias=p),
                dict(out=(r[:5], y))):
        with pytest.raises(N.GlinerDecideError):
            k.block_norm(**{**dict(y=y, residual=r, pre_weight=p), **bad})


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_a_block_over_packed_rows(dtype, kind):
    """Two prompts and a piece through one block, then one more token of each through the same block with the keys
    and values kept: every step against its 64-bit definition on the step's own inputs."""
    kernels = fk()
    C_, H, Hk, D, F = 512, 8, 2, 64, 1024
    w = {name: normal(i, *shape, dtype=dtype, scale=shape[1] ** -0.5) for i, (name, shape) in enumerate(
        dict(qkv=((H + 2 * Hk) * D, C_), out=(C_, H * D), up=(F, C_), down=(C_, F)).items())}
    norms = [(normal(20 + i, C_, dtype=dtype, mean=1.0, scale=0.1),
              normal(30 + i, C_, dtype=dtype, scale=0.1) if kind == "layer" else None) for i in range(4)]
    gate = normal(40, C_, dtype=dtype)

    def block(stream, x, q_lengths, cache, k_lengths):
        qkv = check_projection(x, w["qkv"]).unflatten(1, (H + 2 * Hk, D))
        q, k, v = qkv.split((H, Hk, Hk), dim=1)
        if cache is not None:  # each sequence's kept keys, then its new one
            kept = [torch.cat([torch.cat([c[a:b], t[i:i + 1]]) for i, (a, b) in enumerate(cache[2])])
                    for c, t in zip(cache[:2], (k, v))]
            k, v = kept
        mixed = check_attention(q, k, v, q_lengths, k_lengths)
        y = check_projection(mixed.flatten(1), w["out"])
        stream, x = check_block_norm(y, stream, norms[0], norms[1], gate, 0.7, kind=kind)
        y = check_projection(x, w["up"], None, None, "silu")
        y = check_projection(y, w["down"])
        stream, x = check_block_norm(y, stream, norms[2], norms[3], gate, 0.7, kind=kind)
        return stream, x, k, v

    lengths = [70, 1, 129]
    stream = normal(50, sum(lengths), C_, dtype=torch.float32)
    stream, x, k, v = block(stream, stream.to(dtype), lengths, None, None)
    ends = np.cumsum([0] + lengths)
    spans = [(int(a), int(b)) for a, b in zip(ends[:-1], ends[1:])]
    last = [b - 1 for _, b in spans]
    block(stream[last], x[last], [1, 1, 1], (k, v, spans), [n + 1 for n in lengths])
    # onto the residual stream in the projection's epilogue, in the stream's own memory
    s16 = stream.to(dtype)
    want = check_projection(x, w["up"][:C_], None, s16, "gelu", 0.5)
    assert torch.equal(kernels.projection(x, w["up"][:C_], None, s16, activation="gelu", scale=0.5, out=s16), want)
