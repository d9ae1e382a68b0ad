"""The packed-prompt operators against plain implementations in 64 bits.

Tolerances follow from the arithmetic, per element:
* one rounding to F16 is off by at most 2^-11 of the value (2^-25 among the subnormals);
* an F32 sum of k products on the tensor cores takes k / 16 accumulations, each off by at most
  2^-22 of the sum of magnitudes (aligned addends are cut, not rounded);
* attention's probabilities are rounded to F16 before the second product (tensor-core form),
  which moves an output by at most 2^-11 of sum p |v|, plus n 2^-25 max |v| for those that fall
  among the subnormals."""
from __future__ import annotations

import math

import pytest
import torch

import rustllm_b200 as rb
from rustllm_b200 import _lib

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -11


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def randn(g, *shape, dtype=torch.float16, std=1.0):
    return (torch.randn(shape, generator=g, device=g.device) * std).to(dtype)


def within(got, want, tol):
    """Every element within its tolerance; NaN and infinities have to match."""
    got = got.double()
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.nan_to_num(got[odd], 7.0), torch.nan_to_num(want[odd], 7.0))
    err = torch.where(odd, 0.0, (got - want).abs())
    tol = torch.where(odd, 1.0, tol).clamp(min=1e-300)
    worst = (err / tol).nan_to_num(posinf=1e9, nan=1e9).max() if err.numel() else torch.zeros(())
    assert float(worst) <= 1.0, float(worst)


# ---- batch_tables -----------------------------------------------------------------------
def plain_tables(table, lens, new, bs, nblocks, rows, free=None, start=0):
    table = [list(r) for r in table]
    mb, q_start, pos, seq, slots, used, refused, at = len(table[0]), [0], [], [], [], 0, 0, start
    need_sum = 0
    for s, (c, n) in enumerate(zip(lens, new)):
        n = max(n, 0)
        q_start.append(q_start[-1] + n)
        ok = c >= 0 and c + n <= mb * bs
        need = (-(-(c + n) // bs) - -(-c // bs)) if ok and free is not None else 0
        need_sum += need
        ok = ok and (need == 0 or start + need_sum <= len(free))
        if ok:
            for i in range(need):
                table[s][-(-c // bs) + i] = free[start + need_sum - need + i]
            used += need
        refused += not ok
        for i in range(n):
            p = c + i if ok else -1
            b = table[s][p // bs] if ok else -1
            pos.append(p)
            seq.append(s)
            slots.append(b * bs + p % bs if 0 <= b < nblocks else -1)
    total = q_start[-1]
    over = max(total - rows, 0)
    fill = [-1] * max(rows - total, 0)
    info = [at + used, total, refused, over]
    return (table, q_start, (pos + fill)[:rows], (seq + fill)[:rows], (slots + fill)[:rows], info)


def run_tables(dev, table, lens, new, bs, nblocks, rows, free=None, start=None, out=None):
    t = torch.tensor(table, dtype=torch.int32, device=dev)
    ls = torch.tensor(lens, dtype=torch.int32, device=dev)
    arena = torch.empty((nblocks, 1, bs, 2), dtype=torch.float16, device=dev)
    kv = rb.paged_kv_from_tensors(arena, arena, t, ls)
    fr = None if free is None else torch.tensor(free, dtype=torch.int32, device=dev)
    st = None if start is None else torch.tensor([start], dtype=torch.int32, device=dev)
    nl = torch.tensor(new, dtype=torch.int32, device=dev)
    m = rb.batch_tables(kv, nl, rows, free_blocks=fr, free_start=st, out=out)
    return tuple(x.tolist() for x in (t, *m))


def check_tables(dev, table, lens, new, bs, nblocks, rows, free=None, start=None):
    want = plain_tables(table, lens, new, bs, nblocks, rows, free, start or 0)
    got = run_tables(dev, table, lens, new, bs, nblocks, rows, free, start)
    for w, g, what in zip(want, got, ("table", "q_start", "positions", "row_seq", "slots", "info")):
        assert g == w, what


@pytest.mark.parametrize("seqs,bs,hi,seed", [(1, 16, 1, 0), (7, 16, 40, 1), (64, 8, 1, 2),
                                             (33, 24, 300, 3), (1100, 16, 9, 4), (2500, 5, 3, 5)])
@pytest.mark.parametrize("assign", [True, False])
def test_batch_tables(cuda, seqs, bs, hi, seed, assign):
    import random
    r = random.Random(seed)
    lens = [r.randrange(0, 5 * bs) for _ in range(seqs)]
    new = [r.randint(0 if hi > 1 else 1, hi) for _ in range(seqs)]
    mb = max(-(-(c + n) // bs) for c, n in zip(lens, new)) + 2
    ids = list(range(sum(-(-(c + n) // bs) for c, n in zip(lens, new)) + 9))
    nblocks = len(ids)
    r.shuffle(ids)
    table = [[-1] * mb for _ in range(seqs)]
    for c, n, row in zip(lens, new, table):
        for i in range(-(-c // bs) if assign else -(-(c + n) // bs)):
            row[i] = ids.pop()
    check_tables(cuda, table, lens, new, bs, nblocks, sum(new) + seed, ids if assign else None,
                 3 if assign else None)


def test_batch_tables_refusals_on_the_device(cuda):
    """Negative lengths, tokens past the table, an exhausted free list, unmapped blocks."""
    bs, table = 4, [[9, 8, -1], [7, -1, -1], [-1, -1, -1], [6, 5, 4], [3, -1, -1], [99, 2, -1]]
    lens, new = [8, 2, -1, 10, 4, 5], [1, 2, 5, 3, 6, 3]
    # request 1 fits its block, 2 has a negative length, 3 passes its table, 4 needs 2 blocks
    for free in ([10, 11, 12], [10, 11], [10], []):
        check_tables(cuda, table, lens, new, bs, 16, 24, free)
    check_tables(cuda, table, lens, [-3, 0, 0, 0, 0, 0], bs, 16, 2, [1])
    check_tables(cuda, table, lens, [0] * 6, bs, 16, 0, [1])
    check_tables(cuda, table, lens, new, bs, 16, 24, None)  # -1 and 99 are no blocks: slot -1
    check_tables(cuda, table, lens, new, bs, 16, 7, [10, 11, 12])  # fewer rows than tokens
    check_tables(cuda, table, lens, new, bs, 16, 24, [10, 11, 12], 2)
    # a negative start of the free list (only requests that need no block are placed)
    got = run_tables(cuda, table, lens, new, bs, 16, 24, [10, 11, 12], -1)
    assert got[0] == table and got[5] == [-1, 20, 4, 0]
    assert got[2][1:3] == [2, 3] and got[2][17:20] == [5, 6, 7]
    assert set(got[2][:1] + got[2][3:17] + got[2][20:]) == {-1}
    # a free list holding an id outside the pool: kept in the table, no slot
    check_tables(cuda, table, lens, new, bs, 16, 24, [77, 10, 11])


def test_batch_tables_huge_lengths_saturate(cuda):
    got = run_tables(cuda, [[0], [1], [2]], [0, 0, 0], [2 ** 31 - 1, 2 ** 31 - 1, 1], 16, 4, 5, [3])
    assert got[1] == [0, 2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1]
    assert got[2] == [-1] * 5 and got[3] == [0] * 5 and got[4] == [-1] * 5
    # requests 0 and 1 pass their tables and so need nothing; request 2 takes the one free block
    assert got[0] == [[0], [1], [3]] and got[5] == [1, 2 ** 31 - 1, 2, 2 ** 31 - 1]


def test_batch_tables_again_and_chained(cuda):
    """Calling again changes nothing; the next call's free_start is this call's info[0]."""
    bs, table = 16, torch.full((3, 4), -1, dtype=torch.int32, device=cuda)
    lens = torch.zeros(3, dtype=torch.int32, device=cuda)
    arena = torch.empty((12, 1, bs, 2), dtype=torch.float16, device=cuda)
    kv = rb.paged_kv_from_tensors(arena, arena, table, lens)
    free = torch.arange(12, dtype=torch.int32, device=cuda)
    new = torch.tensor([20, 0, 16], dtype=torch.int32, device=cuda)
    a = rb.batch_tables(kv, new, 40, free_blocks=free)
    first = [x.tolist() for x in (table, *a)]
    b = rb.batch_tables(kv, new, 40, free_blocks=free, out=a)
    assert b is a and [x.tolist() for x in (table, *b)] == first
    lens += new
    c = rb.batch_tables(kv, torch.tensor([13, 1, 0], dtype=torch.int32, device=cuda), 14,
                        free_blocks=free, free_start=a.info[:1])
    assert table.tolist() == [[0, 1, 3, -1], [4, -1, -1, -1], [2, -1, -1, -1]]
    assert c.slots.tolist() == [1 * 16 + 4 + i for i in range(12)] + [3 * 16, 4 * 16]
    assert c.info.tolist() == [5, 14, 0, 0]


# ---- rope_append ------------------------------------------------------------------------
def rotate64(x, pos, cos, sin):
    half = x.shape[-1] // 2
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def append_case(dev, dtype, hq, hkv, d, bs, rows, seed, shift=0, inplace=False, keys=True,
                rope=True):
    g = gen(dev, seed)
    w = (hq + 2 * hkv) * d + (8 if shift == 0 else 3)  # fused rows with a tail
    buf = randn(g, rows * w + 8, dtype=dtype)[shift:shift + rows * w].view(rows, w)
    q, k = buf[:, :hq * d].unflatten(1, (hq, d)), buf[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    v = buf[:, (hq + hkv) * d:(hq + 2 * hkv) * d].unflatten(1, (hkv, d))
    nblocks = rows // bs + 3
    kc, vc = (randn(g, nblocks, hkv, bs, d, dtype=dtype) for _ in range(2))
    kv = rb.paged_kv_from_tensors(kc, vc, torch.zeros((1, 1), dtype=torch.int32, device=dev),
                                  torch.zeros(1, dtype=torch.int32, device=dev))
    pos = torch.randint(0, 500, (rows,), generator=g, device=dev, dtype=torch.int32)
    slots = torch.randperm(nblocks * bs, generator=g, device=dev)[:rows].contiguous()
    if rows > 4:
        pos[1], pos[3] = -1, 499
        slots[2], slots[4] = -1, nblocks * bs  # outside the arena: not cached
    cos, sin = rb.rope_tables(d, 499, 10000.0, device=dev)  # position 499 is past the table
    x, y, z = (t.clone() for t in (q, k, v))
    ck, cv = kc.clone(), vc.clone()
    qo = q if inplace else torch.full((rows, hq, d), 5.0, dtype=dtype, device=dev)
    ko = (k if inplace else torch.full((rows, hkv, d), 5.0, dtype=dtype, device=dev)) if keys else None
    rb.rope_append(kv, q, k, v, pos, slots, rope=(cos, sin) if rope else None, q_out=qo, k_out=ko)
    p = pos.long()
    live, turn = p >= 0, (p >= 0) & (p < 499)

    def want(t, old):
        r = rotate64(t, p.clamp(0, 498), cos, sin)
        r = torch.where((turn if rope else torch.zeros_like(turn))[:, None, None], r, t.double())
        return torch.where(live[:, None, None], r, old.double())

    half = HALF if dtype == torch.float16 else 2.0 ** -24

    def tol(t, r):  # two products and a sum in F32, then the storage rounding
        m = t.double().abs()
        m = m + m.roll(d // 2, -1)
        return half * r.abs() + 2.0 ** -22 * m + 2.0 ** -25

    wq, wk = want(x, x if inplace else torch.full_like(x, 5.0)), want(y, y if inplace else torch.full_like(y, 5.0))
    within(qo, wq, tol(x, wq))
    if keys:
        within(ko, wk, tol(y, wk))
    sl = torch.where(live, slots, -1)
    put = (sl >= 0) & (sl < nblocks * bs)
    fk, fv = ck.double().transpose(1, 2).reshape(-1, hkv, d), cv.transpose(1, 2).reshape(-1, hkv, d)
    rk = want(y, y)
    fk[sl[put]] = rk[put]
    fv[sl[put]] = z[put]
    gk, gv = kc.transpose(1, 2).reshape(-1, hkv, d), vc.transpose(1, 2).reshape(-1, hkv, d)
    bound = torch.zeros_like(fk)
    bound[sl[put]] = tol(y, rk)[put]
    within(gk, fk, bound)
    assert torch.equal(gv, fv)
    if keys:  # the cached keys are the dense ones, bit for bit
        assert torch.equal(gk[sl[put]], ko[put])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d,bs", [(9, 3, 64, 16), (32, 8, 128, 16), (5, 5, 80, 24),
                                         (4, 1, 96, 8), (6, 2, 32, 1), (2, 1, 256, 16),
                                         (3, 3, 6, 7), (2, 2, 2, 4), (1, 1, 600, 4)])
@pytest.mark.parametrize("rows", [1, 70])
def test_rope_append(cuda, dtype, hq, hkv, d, bs, rows):
    append_case(cuda, dtype, hq, hkv, d, bs, rows, seed=d + rows)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rope_append_forms(cuda, dtype):
    append_case(cuda, dtype, 9, 3, 64, 16, 40, 1, inplace=True)
    append_case(cuda, dtype, 9, 3, 64, 16, 40, 2, keys=False)
    append_case(cuda, dtype, 9, 3, 64, 16, 40, 3, rope=False)
    append_case(cuda, dtype, 9, 3, 64, 16, 40, 4, shift=1)  # rows off the 16-byte grid
    append_case(cuda, dtype, 32, 8, 128, 16, 5000, 5, inplace=True)


def test_rope_append_new_output_is_zero_in_padding(cuda):
    q = torch.ones(3, 2, 8, dtype=torch.float16, device=cuda)
    c = torch.zeros(2, 2, 4, 8, dtype=torch.float16, device=cuda)
    kv = rb.paged_kv_from_tensors(c, c.clone(), torch.zeros((1, 1), dtype=torch.int32, device=cuda),
                                  torch.zeros(1, dtype=torch.int32, device=cuda))
    pos = torch.tensor([0, -1, 5], dtype=torch.int32, device=cuda)
    slots = torch.tensor([7, 2, -1], device=cuda)
    out, none = rb.rope_append(kv, q, q, q, pos, slots)
    assert none is None and out[1].abs().sum() == 0 and bool((out[[0, 2]] == 1).all())
    assert c[1, :, 3].eq(1).all() and c.sum() == 16


def test_rope_append_matches_the_prefill_cache(cuda):
    """batch_tables + rope_append leave the cache as the prefill call leaves it."""
    g = gen(cuda, 5)
    lens, hq, hkv, d = [37, 0, 5, 64], 4, 2, 64
    a, b = (rb.PagedKvCache(1, 4, 100, hkv, d, shuffle_seed=3, device=cuda) for _ in range(2))
    old = randn(g, hkv, 21, d)
    for c in (a, b):
        c.append(0, 2, old, old)
        c.advance(21, 2)
        for s, n in enumerate(lens):
            c.reserve(s, n)
    rows = sum(lens)
    q, k, v = randn(g, rows, hq, d), randn(g, rows, hkv, d), randn(g, rows, hkv, d)
    rope = rb.rope_tables(d, 200, 10000.0, device=cuda)
    m = rb.batch_tables(a.view(0), torch.tensor(lens, dtype=torch.int32, device=cuda), rows)
    rb.rope_append(a.view(0), q, k, v, m.positions, m.slots, rope=rope)
    rb.gqa_prefill(b.view(0), q, k, v, q_start=m.q_start, rope=rope)
    for c in (a, b):
        for s, n in enumerate(lens):
            c.advance(n, s)
    for s in range(4):
        for x, y in zip(a.gather(0, s), b.gather(0, s)):
            assert torch.equal(x, y)


# ---- prompt_attention -------------------------------------------------------------------
def plain_attention(q, k, v, starts, scale):
    """(out, lse, sum p |v|, largest sum |q||k| scale) per row in 64 bits; only visible keys are
    ever read."""
    rows, hq, d = q.shape
    g = hq // k.shape[1]
    out, lse = torch.zeros(rows, hq, d).double(), torch.zeros(rows, hq).double()
    mag, dot = torch.zeros(rows, hq, d).double(), 0.0
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    for lo, hi in zip(starts, starts[1:]):
        for h in range(hq):
            s = q[lo:hi, h] @ k[lo:hi, h // g].T * scale
            a = q[lo:hi, h].abs() @ k[lo:hi, h // g].abs().T * scale
            if a.numel():
                dot = max(dot, float(a.nan_to_num(0, 0, 0).max()))
            vis = torch.ones_like(s, dtype=torch.bool).tril()
            s = torch.where(vis, s, -math.inf)
            m = s.max(-1, keepdim=True).values if s.numel() else s
            m0 = torch.where(m == -math.inf, 0.0, m) if s.numel() else m
            p = torch.where(vis, torch.exp(s - m0), 0.0)
            l = p.sum(-1, keepdim=True)
            w = torch.where(l == 0, 0.0, p / l)
            x = v[lo:hi, h // g]
            if torch.isfinite(x).all():
                out[lo:hi, h], mag[lo:hi, h] = w @ x, w @ x.abs()
            else:  # masked values are skipped, not multiplied by zero
                for i in range(hi - lo):
                    out[lo + i, h] = w[i, :i + 1] @ x[:i + 1]
                    mag[lo + i, h] = w[i, :i + 1] @ x[:i + 1].abs()
            lse[lo:hi, h] = (m0 + torch.log(l))[:, 0] if s.numel() else 0
    return out, lse, mag, dot


def attention_case(dev, lens, hq, hkv, d, dtype=torch.float16, seed=0, pad=0, scale=0.0,
                   out_dtype=None, lead=0, spoil=None, std=1.0, max_rows=None, inplace=False,
                   shift=0):
    g = gen(dev, seed)
    starts = [lead]
    for n in lens:
        starts.append(starts[-1] + n)
    rows = starts[-1] + pad
    w = (hq + 2 * hkv) * d
    x = randn(g, rows * w + 16, dtype=dtype, std=std)[shift:shift + rows * w].view(rows, w)
    q = x[:, :hq * d].unflatten(1, (hq, d))
    k = x[:, hq * d:(hq + hkv) * d].unflatten(1, (hkv, d))
    v = x[:, (hq + hkv) * d:].unflatten(1, (hkv, d))
    if spoil:
        spoil(q, k, v, starts)
    sc = scale if scale > 0 else d ** -0.5
    want, wl, mag, dot = plain_attention(q, k, v, starts, sc)
    if inplace:
        q = q.contiguous()
    out = q if inplace else torch.full((rows, hq, d), 9.0, dtype=out_dtype or dtype, device=dev)
    before = out.clone()
    lse = torch.full((rows, hq), 9.0, device=dev)
    qs = torch.tensor(starts, dtype=torch.int32, device=dev)
    rb.prompt_attention(q, k, v, qs, max(lens) if max_rows is None else max_rows, scale=scale,
                        out=out, lse=lse)
    torch.cuda.synchronize()
    assert rb.prompt_status() == 0
    lo, hi = starts[0], starts[-1]
    assert torch.equal(out[:lo], before[:lo]) and torch.equal(out[hi:], before[hi:])
    assert bool((lse[:lo] == 9).all()) and bool((lse[hi:] == 9).all())
    n = max(lens)
    eps = HALF if out.dtype == torch.float16 else 2.0 ** -24
    f16 = dtype == torch.float16
    # scores: F32 sums of d products (tensor cores: d / 16 steps), then exp2 of a rounded
    # difference of values up to `dot`
    score = ((d / 16 + 2) * 2.0 ** -22 if f16 else d * 2.0 ** -24) * dot + 2.0 ** -22 * (dot + 2)
    rel = 2 * score + ((HALF if f16 else 0) + (n + 8) * 2.0 ** -24 + 2.0 ** -21)
    vmax = float(v[lo:hi].double().nan_to_num(0, 0, 0).abs().max()) if hi > lo else 0
    tol = eps * want.abs() + rel * mag.nan_to_num(0, 0, 0) + 2.0 ** -25 + (
        n * 2.0 ** -25 * vmax if f16 else 0)
    within(out[lo:hi].cpu(), want[lo:hi], tol[lo:hi])
    within(lse[lo:hi].cpu(), wl[lo:hi], 2.0 ** -22 * wl[lo:hi].abs().nan_to_num(0, 0, 0) + score +
           2.0 ** -20)
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("hq,hkv,d", [(9, 3, 64), (4, 1, 128), (3, 3, 64), (2, 1, 32), (2, 2, 80),
                                      (5, 5, 96), (2, 1, 8), (2, 1, 256), (1, 1, 7), (4, 2, 136)])
def test_prompt_attention(cuda, dtype, hq, hkv, d):
    attention_case(cuda, [1, 0, 37, 130, 64, 2], hq, hkv, d, dtype, seed=d, pad=3, lead=2)


@pytest.mark.parametrize("lens", [[1], [32], [127], [128], [129], [255, 1, 257], [0, 0, 5, 0],
                                  [1] * 40, [300, 513], [640]])
@pytest.mark.parametrize("hq,hkv,d", [(6, 2, 64), (4, 4, 128), (8, 1, 128), (3, 1, 64)])
def test_prompt_attention_lengths(cuda, lens, hq, hkv, d):
    attention_case(cuda, lens, hq, hkv, d, seed=len(lens) + d, pad=len(lens) % 3)


def test_prompt_attention_f32_lengths(cuda):
    for lens in ([1], [63, 64, 65], [0, 200]):
        attention_case(cuda, lens, 9, 3, 64, torch.float32, seed=3)


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (torch.float32, 40), (torch.float32, 128),
                                     (torch.float32, 200), (torch.float16, 20), (torch.float16, 136)])
def test_prompt_attention_cuda_cores_many_heads(cuda, dtype, d):
    """Enough heads for 64 rows a CTA (32 rows and two teams a CTA otherwise), the keys that rows
    do not see not finite."""
    lens = [1, 63, 130, 0, 65, 200]
    attention_case(cuda, lens, 48, 4, d, dtype, seed=d, pad=3, lead=2)

    def spoil(q, k, v, starts):
        end = starts[-1]
        k[end:], v[end:], q[end:], k[:2], v[:2] = (math.nan,) * 5
        k[end - 30], v[end - 30], v[end - 1] = math.nan, math.inf, -math.inf
    attention_case(cuda, lens, 48, 4, d, dtype, seed=d + 1, pad=3, lead=2, spoil=spoil)


@pytest.mark.parametrize("d", [64, 24, 128])
@pytest.mark.parametrize("n", [64, 65, 96, 97, 128, 129, 160, 193, 320])
def test_prompt_attention_cuda_cores_tiles(cuda, d, n):
    """One sequence ending before, at and behind the tiles of 64 keys that two teams take in turn."""
    attention_case(cuda, [n], 2, 1, d, torch.float32, seed=n, std=2.0)
    out = attention_case(cuda, [n, 3], 2, 1, d, torch.float32, seed=n,
                         spoil=lambda q, k, v, s: (q.abs_(), k[:n - 1].fill_(-math.inf)))
    assert bool((out[:n - 1] == 0).all()) and bool((out[n - 1] != 0).any())


def test_prompt_attention_long(cuda):
    attention_case(cuda, [2000, 100, 1100], 3, 1, 64, seed=1)
    attention_case(cuda, [1500], 2, 1, 128, seed=2)


@pytest.mark.parametrize("lens", [[1], [129], [255, 1, 257], [0, 0, 5, 0], [1] * 40, [70, 200, 300]])
@pytest.mark.parametrize("hq,hkv,d", [(6, 2, 64), (3, 1, 64), (2, 2, 40)])
def test_prompt_attention_few_long_sequences(cuda, lens, hq, hkv, d):
    """Room for 1024 rows a sequence: heads up to 64 go in steps of 128 keys instead of 64."""
    attention_case(cuda, lens, hq, hkv, d, seed=d, lead=3, pad=1024 * len(lens) - sum(lens))

    def spoil(q, k, v, starts):
        end = starts[-1]
        k[end:], v[end:], q[end:] = math.nan, math.nan, math.nan
        k[:3], v[:3] = math.nan, math.inf
        v[end - 1] = math.inf
    attention_case(cuda, lens, hq, hkv, d, seed=d, lead=3, pad=1024 * len(lens), spoil=spoil)


def test_prompt_attention_many_rows(cuda):
    """More packed rows than one launch schedules (131,072), tiles shared by two or three
    sequences, and one sequence across the border."""
    attention_case(cuda, [100] * 1305 + [900] + [77] * 60, 1, 1, 32, seed=1, pad=40)
    attention_case(cuda, [60] * 2190, 2, 1, 72, seed=2)


def test_prompt_attention_forms(cuda):
    attention_case(cuda, [70, 200], 4, 2, 64, out_dtype=torch.float32, seed=1)
    attention_case(cuda, [70, 200], 4, 2, 64, scale=0.7, seed=2)     # sharp rows
    attention_case(cuda, [70, 200], 4, 2, 128, std=4.0, seed=3)      # scores in the hundreds
    attention_case(cuda, [70, 200], 4, 2, 64, max_rows=1000, seed=4)
    attention_case(cuda, [70, 200], 4, 2, 64, inplace=True, seed=5)
    attention_case(cuda, [70, 200], 4, 2, 128, inplace=True, seed=6)
    attention_case(cuda, [70, 200], 4, 2, 64, shift=1, seed=7)       # off the 16-byte grid
    attention_case(cuda, [70, 200], 4, 2, 64, torch.float32, inplace=True, seed=8)
    attention_case(cuda, [200] * 70, 2, 1, 64, seed=9)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 128])
def test_prompt_attention_hidden_values_never_matter(cuda, dtype, d):
    """NaN and infinities in keys and values that a row does not see, in its own sequence, in
    its neighbours and in padding, leave the row's result alone; where it sees them they show."""
    def spoil(q, k, v, starts):
        a, b, c = starts[1], starts[2], starts[3]
        k[a + 100:a + 104], v[a + 100] = math.nan, math.inf    # in the middle of a sequence
        v[a + 150, :, 3], v[a + 151, :, 3] = -math.inf, math.nan
        v[a + 199] = math.inf                                  # its last row
        v[b + 5, :, 7], v[b + 6, :, 8] = math.inf, -math.inf   # and of the next one
        k[c:], v[c:] = math.nan, math.nan                      # padding
        q[c:] = math.nan
        k[:starts[0]], v[:starts[0]] = math.nan, math.nan
    attention_case(cuda, [70, 200, 300], 2, 1, d, dtype, seed=d, pad=9, lead=5, spoil=spoil)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_prompt_attention_infinite_scores(cuda, dtype):
    """A row whose visible scores are all -inf gives zeros (softmax of the framework)."""
    def spoil(q, k, v, starts):
        q[:] = q.abs()
        k[starts[0]:starts[0] + 3] = -math.inf
    out = attention_case(cuda, [40, 20], 2, 1, 64, dtype, seed=3, spoil=spoil)
    assert bool((out[:3] == 0).all()) and bool((out[3:] != 0).any())


# ---- prompt_linear ----------------------------------------------------------------------
def linear_case(dev, rows, k, n, act="none", bias=False, residual=False, xpad=0, seed=0,
                inplace=False, opad=0, wpad=0):
    g = gen(dev, seed)
    wide = 2 * n if act == "swiglu" else n
    x = randn(g, rows, k + xpad)[:, :k]
    w = randn(g, k, wide + wpad, std=1 / math.sqrt(k))[:, :wide]
    b = randn(g, wide, std=0.5) if bias else None
    res = randn(g, rows, n + opad)[:, :n] if residual else None
    r64 = res.double() if residual else torch.zeros((), device=dev).double()
    out = res if inplace else torch.full((rows, n + opad), 3.0, dtype=torch.float16,
                                         device=dev)[:, :n]
    got = rb.prompt_linear(x, w, bias=b, activation=act, residual=res, out=out)
    assert got is out
    torch.cuda.synchronize()
    assert rb.prompt_status() == 0
    y, mag = x.double() @ w.double(), x.double().abs() @ w.double().abs()
    if bias:
        y, mag = y + b.double(), mag + b.double().abs()
    e = (k / 16 + 4) * 2.0 ** -22 * mag
    if act == "swiglu":
        gate, up, eg, eu = y[:, :n], y[:, n:], e[:, :n], e[:, n:]
        s = gate * torch.sigmoid(gate)
        want, err = s * up, 1.1 * eg * up.abs() + s.abs() * eu + 2.0 ** -19 * (s * up).abs()
    else:
        f = dict(none=lambda t: t, relu=lambda t: t.clamp(min=0), gelu=lambda t: t * torch.special.ndtr(t),
                 silu=lambda t: t * torch.sigmoid(t))[act]
        want, err = f(y), 1.13 * e + 2.0 ** -19 * f(y).abs()
    want = want + r64
    within(out, want, HALF * want.abs() + err + 2.0 ** -24 * (want.abs() + r64.abs()) + 2.0 ** -25)
    if opad and not inplace:  # columns beside the result
        full = torch.as_strided(out, (rows, n + opad), (n + opad, 1))
        assert bool((full[:, n:] == 3).all())


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "swiglu"])
@pytest.mark.parametrize("rows,k,n", [(1, 64, 64), (33, 768, 200), (129, 72, 520), (300, 576, 264)])
def test_prompt_linear(cuda, act, rows, k, n):
    linear_case(cuda, rows, k, n, act, bias=True, residual=True, seed=rows)
    linear_case(cuda, rows, k, n, act, seed=rows + 1)


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 64, 65, 127, 128, 129, 257, 1000])
@pytest.mark.parametrize("k,n", [(8, 8), (768, 2304), (2560, 960), (136, 136)])
def test_prompt_linear_sizes(cuda, rows, k, n):
    linear_case(cuda, rows, k, n, bias=True, seed=rows)


def test_prompt_linear_strides_and_place(cuda):
    linear_case(cuda, 70, 320, 256, xpad=8, opad=24, wpad=64, residual=True, seed=1)
    linear_case(cuda, 300, 320, 264, xpad=64, residual=True, inplace=True, seed=2)
    linear_case(cuda, 40, 320, 264, "swiglu", residual=True, inplace=True, opad=8, seed=3)
    linear_case(cuda, 5000, 256, 1024, "silu", bias=True, residual=True, seed=4)
    linear_case(cuda, 4097, 512, 520, "swiglu", bias=True, seed=5)


@pytest.mark.parametrize("rows,k,n", [(2304, 264, 2048), (2049, 72, 2040), (16640, 64, 256)])
def test_prompt_linear_pairs_of_ctas(cuda, rows, k, n):
    """Sizes whose tiles fit one wave of CTA pairs, with a last pair that is not full."""
    linear_case(cuda, rows, k, n, "gelu", bias=True, seed=1)
    linear_case(cuda, rows, k, n, residual=True, inplace=True, seed=2)
    linear_case(cuda, rows, k, n // 2 + 8 - n // 2 % 8, "swiglu", bias=True, residual=True, seed=3)


@pytest.mark.parametrize("rows,k,n,act", [
    (33, 4096, 64, "none"), (1, 4104, 88, "gelu"), (130, 4096, 512, "relu"), (33, 4040, 1000, "silu"),
    (512, 1024, 1024, "none"), (256, 4096, 4096, "gelu"), (33, 4096, 4096, "none"),
    (33, 8192, 1016, "silu"), (33, 4096, 2048, "swiglu"), (9, 2048, 2560, "swiglu"),
    (70, 4104, 488, "swiglu"), (129, 520, 40, "none"), (300, 4096, 4088, "gelu"),
    (500, 4104, 4096, "none"), (300, 4096, 2040, "swiglu")])
def test_prompt_linear_long_products_of_few_tiles(cuda, rows, k, n, act):
    """K split over 2, 4 and 8 CTAs, columns and K that no part divides."""
    linear_case(cuda, rows, k, n, act, bias=True, residual=True, seed=rows, xpad=8, opad=8, wpad=16)
    linear_case(cuda, rows, k, n, act, seed=rows + 1)
    linear_case(cuda, rows, k, n, act, residual=True, seed=rows + 2, inplace=True)


def test_prompt_linear_split_again_and_captured(cuda):
    """The same bits every time, also from a replayed graph beside another stream's calls."""
    g = gen(cuda, 5)
    x, w = randn(g, 40, 4096), randn(g, 4096, 600, std=1 / 64)
    want = rb.prompt_linear(x, w, activation="gelu")
    out, other = torch.empty_like(want), torch.empty_like(want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rb.prompt_linear(x, w, activation="gelu", out=out)
    side = torch.cuda.Stream()
    for _ in range(20):
        graph.replay()
        with torch.cuda.stream(side):
            rb.prompt_linear(x, w, activation="gelu", out=other)
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(other, want) and rb.prompt_status() == 0


def test_prompt_linear_non_finite_rows_stay_apart(cuda):
    """NaN in one row of x, or past k in its buffer, reaches that row alone."""
    x = torch.ones(200, 128, dtype=torch.float16, device=cuda)
    x[:, 64:] = math.nan
    x[77, 3] = math.inf
    w = torch.full((64, 72), 0.5, dtype=torch.float16, device=cuda)
    y = rb.prompt_linear(x[:, :64], w)
    assert bool((y[77] == math.inf).all())
    keep = torch.arange(200, device=cuda) != 77
    assert bool((y[keep] == 32).all())


def test_prompt_linear_overflow_is_inf(cuda):
    x = torch.full((3, 64), 300.0, dtype=torch.float16, device=cuda)
    y = rb.prompt_linear(x, torch.full((64, 8), 30.0, dtype=torch.float16, device=cuda))
    assert bool((y == math.inf).all())


# ---- refusals of the Python layer -------------------------------------------------------
def test_python_refusals(cuda):
    h = dict(dtype=torch.float16, device=cuda)
    q, k, w = torch.zeros(4, 4, 64, **h), torch.zeros(4, 2, 64, **h), torch.zeros(64, 128, **h)
    st = torch.tensor([0, 4], dtype=torch.int32, device=cuda)
    x = torch.zeros(4, 64, **h)
    for bad in (k.float(), k.cpu(), k[:3], k[..., :32], k.transpose(0, 1), k[:1].expand(4, 2, 64)):
        with pytest.raises(rb.TinyError):
            rb.prompt_attention(q, bad, k, st, 4)
        with pytest.raises(rb.TinyError):
            rb.prompt_attention(q, k, bad, st, 4)
    for kw in (dict(q_start=st.long()), dict(q_start=st[:1]), dict(max_rows=-1),
               dict(out=torch.zeros(4, 4, 64, device=cuda, dtype=torch.float64)),
               dict(out=torch.zeros(4, 8, 64, **h)[:, ::2]), dict(lse=torch.zeros(4, 3, device=cuda))):
        with pytest.raises(rb.TinyError):
            rb.prompt_attention(**{**dict(q=q, k=k, v=k, q_start=st, max_rows=4), **kw})
    for kw in (dict(x=x.float()), dict(w=w.t()), dict(w=w[:32]), dict(bias=torch.zeros(64, **h)),
               dict(bias=torch.zeros(128, device=cuda)), dict(activation="tanh"),
               dict(residual=torch.zeros(3, 128, **h)), dict(residual=torch.zeros(1, 128, **h).expand(4, 128)),
               dict(out=torch.zeros(4, 64, **h)), dict(w=w[:, :60]), dict(x=x[:, 1:9], w=w[:8]),
               dict(w=torch.zeros(64, 31, **h), activation="swiglu")):
        with pytest.raises(rb.TinyError):
            rb.prompt_linear(**{**dict(x=x, w=w), **kw})
    arena = torch.zeros(4, 2, 16, 64, **h)
    lens = torch.zeros(1, dtype=torch.int32, device=cuda)
    kv = rb.paged_kv_from_tensors(arena, arena, torch.zeros((1, 4), dtype=torch.int32, device=cuda), lens)
    for a in ((lens.long(), 4), (lens.expand(2), 4), (lens, -1), (lens.cpu(), 4)):
        with pytest.raises(rb.TinyError):
            rb.batch_tables(kv, *a)
    with pytest.raises(rb.TinyError):
        rb.batch_tables(kv, lens, 4, free_start=lens)
    with pytest.raises(rb.TinyError):
        rb.batch_tables(kv, lens, 4, out=rb.BatchTables.empty(1, 5, cuda))
    p, s = torch.zeros(4, dtype=torch.int32, device=cuda), torch.zeros(4, dtype=torch.int64, device=cuda)
    cos = torch.zeros(8, 32, device=cuda)
    for kw in (dict(positions=p.long()), dict(slots=p), dict(slots=s[:3]), dict(k=k[:, :1]),
               dict(v=k.float()), dict(rope=(cos[:, :16], cos)), dict(rope=(cos.half(), cos)),
               dict(q_out=q[:3]), dict(k_out=q), dict(q=q[..., :32])):
        with pytest.raises(rb.TinyError):
            rb.rope_append(**{**dict(kv=kv, q=q, k=k, v=k, positions=p, slots=s), **kw})
    assert float(arena.abs().sum()) == 0


# ---- streams, graphs, repeats -----------------------------------------------------------
def chain(dev, w, lens, table, arena, free, bufs):
    """Maps, projection, append, attention, projection: one packed layer."""
    kv = rb.paged_kv_from_tensors(*arena, table, bufs["cached"])
    m = rb.batch_tables(kv, lens, bufs["x"].shape[0], free_blocks=free, out=bufs["maps"])
    hq, hkv, d = 4, 2, 64
    rb.prompt_linear(bufs["x"], w["qkv"], bias=w["b"], out=bufs["qkv"])
    f = bufs["qkv"]
    q, k, v = (f[:, a * d:b * d].unflatten(1, (b - a, d)) for a, b in
               ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    rb.rope_append(kv, q, k, v, m.positions, m.slots, rope=w["rope"], q_out=q, k_out=k)
    rb.prompt_attention(q, k, v, m.q_start, bufs["max"], out=bufs["attn"])
    return rb.prompt_linear(bufs["attn"].flatten(1), w["o"], residual=bufs["x"], out=bufs["y"])


def chain_setup(dev, lens, seed=0):
    g = gen(dev, seed)
    rows = sum(lens) + 5
    w = dict(qkv=randn(g, 256, 512, std=0.06), b=randn(g, 512, std=0.1), o=randn(g, 256, 256, std=0.06),
             rope=rb.rope_tables(64, 600, 10000.0, device=dev))
    n = sum(-(-x // 16) for x in lens)
    arena = (torch.zeros(n + 2, 2, 16, 64, dtype=torch.float16, device=dev),
             torch.zeros(n + 2, 2, 16, 64, dtype=torch.float16, device=dev))
    table = torch.full((len(lens), 40), -1, dtype=torch.int32, device=dev)
    free = torch.randperm(n + 2, generator=g, device=dev).int()
    bufs = dict(x=randn(g, rows, 256), qkv=torch.zeros(rows, 512, dtype=torch.float16, device=dev),
                attn=torch.zeros(rows, 4, 64, dtype=torch.float16, device=dev),
                y=torch.zeros(rows, 256, dtype=torch.float16, device=dev), max=max(lens),
                cached=torch.zeros(len(lens), dtype=torch.int32, device=dev),
                maps=rb.BatchTables.empty(len(lens), rows, dev))
    return w, torch.tensor(lens, dtype=torch.int32, device=dev), table, arena, free, bufs


def test_chain_against_64_bits_and_captured(cuda):
    """The four operators as a layer runs them: against 64 bits, bit-identical on repeats, on
    another stream, and in a captured graph replayed on new inputs."""
    lens = [37, 1, 0, 200, 16]
    w, new, table, arena, free, bufs = chain_setup(cuda, lens)
    y = chain(cuda, w, new, table, arena, free, bufs).clone()
    rows, total = bufs["x"].shape[0], sum(lens)
    # 64 bits on the stored F16 intermediates: each step has its own rounding
    f = bufs["qkv"].double()
    want = bufs["attn"].flatten(1).double() @ w["o"].double() + bufs["x"].double()
    tol = HALF * want.abs() + 24 * 2.0 ** -22 * (
        bufs["attn"].flatten(1).double().abs() @ w["o"].double().abs() + bufs["x"].double().abs()) + 2.0 ** -25
    within(y, want, tol)
    q, k, v = (f[:, a:b].view(rows, -1, 64) for a, b in ((0, 256), (256, 384), (384, 512)))
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    o, _, mag, dot = plain_attention(q.half(), k.half(), v.half(), starts, 0.125)
    atol = HALF * o.abs() + (HALF + 40 * 2.0 ** -22 * (dot + 2) + 300 * 2.0 ** -24) * mag + 200 * 2.0 ** -25 * 8
    within(bufs["attn"][:total].cpu(), o[:total], atol[:total])
    assert bool((bufs["attn"][total:] == 0).all())
    # the cache holds the rotated keys and the values
    sl = bufs["maps"].slots[:total]
    for a, t in zip(arena, (k, v)):
        flat = a.transpose(1, 2).reshape(-1, 2, 64)
        assert torch.equal(flat[sl], t[:total].half())
    assert torch.equal(y, chain(cuda, w, new, table, arena, free, bufs))
    side = torch.cuda.Stream(cuda)
    side.wait_stream(torch.cuda.current_stream(cuda))
    with torch.cuda.stream(side):
        again = chain(cuda, w, new, table, arena, free, bufs).clone()
    torch.cuda.current_stream(cuda).wait_stream(side)
    assert torch.equal(y, again)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain(cuda, w, new, table, arena, free, bufs)
    # other inputs and other lengths (within max and rows) through the same graph
    other = [120, 0, 64, 3, 50]
    bufs["x"].copy_(randn(gen(cuda, 9), rows, 256))
    new.copy_(torch.tensor(other, dtype=torch.int32))
    table.fill_(-1)
    bufs["attn"].zero_()
    graph.replay()
    replayed = [t.clone() for t in (bufs["y"], table, *bufs["maps"])]
    table.fill_(-1)
    bufs["attn"].zero_()
    chain(cuda, w, new, table, arena, free, bufs)
    for a, b in zip(replayed, (bufs["y"], table, *bufs["maps"])):
        assert torch.equal(a, b)
    assert rb.prompt_status() == 0


def test_two_streams_at_once(cuda):
    """Independent calls on two streams share no state."""
    lens = [300, 41, 7]
    jobs = [chain_setup(cuda, lens, seed=s) for s in (1, 2)]
    alone = [chain(cuda, *j).clone() for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda) for _ in jobs]
    for j in jobs:
        j[-1]["y"].zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for st, j in zip(streams, jobs):
            with torch.cuda.stream(st):
                chain(cuda, *j)
    torch.cuda.synchronize()
    for j, y in zip(jobs, alone):
        assert torch.equal(j[-1]["y"], y)


# ---- the decoder's packed prefill -------------------------------------------------------
def packed_decoder(dev, seqs, seed=3, hidden=256, heads=4, kv=2, inter=512, max_len=400):
    from rustllm_b200.decoder import Decoder, DecoderWeights, ModelConfig
    cfg = ModelConfig(vocab_size=1000, hidden_size=hidden, intermediate_size=inter, num_layers=2,
                      num_heads=heads, num_kv_heads=kv, max_seq_len=max_len, rms_norm_eps=1e-5,
                      rope_theta=10000.0)
    w = DecoderWeights(cfg, device=dev, seed=seed, std=0.05)
    return cfg, w, Decoder(cfg, w, seqs, device=dev, shuffle_seed=7)


def prompt_ids(dev, lens, seed=0):
    g = gen(dev, seed)
    return [torch.randint(0, 1000, (n,), generator=g, device=dev) for n in lens]


def close_logits(got, want):
    """A few F16 layers against another order of the same roundings (as the decoder's own
    tests): 3e-2 of the largest logit."""
    got, want = got.double(), want.double()
    assert float((got - want).abs().max()) <= 3e-2 * float(want.abs().max())


@pytest.mark.parametrize("lens,hidden,heads,kv", [([37, 1, 200, 16], 256, 4, 2),
                                                  ([5, 130], 576, 9, 3), ([300], 512, 4, 4)])
def test_decoder_prefill_packed(cuda, lens, hidden, heads, kv):
    """Logits after ragged prompts against the float32 model, the cache and decode steps behind
    them against prompts run token by token."""
    from model_reference import reference_forward
    cfg, w, dec = packed_decoder(cuda, len(lens), hidden=hidden, heads=heads, kv=kv)
    prompts = prompt_ids(cuda, lens)
    first = dec.prefill_packed(prompts)
    assert dec.cache.lens() == lens and rb.prompt_status() == 0
    for s, p in enumerate(prompts):
        close_logits(dec.logits[s], reference_forward(cfg, w, p)[-1])
    assert torch.equal(first, dec.next_ids)
    tokens = dec.decode(3, first)
    # the same prompts one sequence at a time, through the equal-length prefill
    for s, p in enumerate(prompts):
        _, _, one = packed_decoder(cuda, 1, hidden=hidden, heads=heads, kv=kv)
        one.prefill(p[None])
        for li in range(cfg.num_layers):
            for a, b in zip(dec.cache.gather(li, s), one.cache.gather(li, 0)):
                n = lens[s]
                err = (a[:, :n].double() - b[:, :n].double()).abs().max()
                assert float(err) <= 2e-2 * float(b.double().abs().max())
    # and the steps behind them follow the full model on prompt + tokens
    full = torch.cat([prompts[0], torch.stack([first[0], *tokens[:2, 0]]).long()])
    close_logits(dec.logits[0], reference_forward(cfg, w, full)[-1])


def test_decoder_prefill_packed_behind_cached_tokens(cuda):
    """A second ragged batch attends what the first one cached (the paged path)."""
    from model_reference import reference_forward
    cfg, w, dec = packed_decoder(cuda, 3)
    a, b = prompt_ids(cuda, [20, 3, 150], 1), prompt_ids(cuda, [1, 140, 30], 2)
    dec.prefill_packed(a)
    dec.prefill_packed(b)
    assert dec.cache.lens() == [21, 143, 180]
    for s in range(3):
        close_logits(dec.logits[s], reference_forward(cfg, w, torch.cat([a[s], b[s]]))[-1])


def test_decoder_prefill_packed_refusals(cuda):
    _, _, dec = packed_decoder(cuda, 2, max_len=32)
    ids = prompt_ids(cuda, [3, 4])
    with pytest.raises(rb.ShapeMismatch):
        dec.prefill_packed(ids[:1])
    with pytest.raises(rb.InvalidShape):
        dec.prefill_packed([ids[0], ids[1][:0]])
    with pytest.raises(rb.InvalidShape):
        dec.prefill_packed([ids[0], ids[1][None]])
    with pytest.raises(rb.PositionOutOfRange):
        dec.prefill_packed([ids[0], torch.zeros(33, dtype=torch.int64, device=cuda)])
    with pytest.raises(rb.InvalidArgument):
        dec.prefill_packed([ids[0], torch.full((2,), 1000, device=cuda)])
    assert dec.cache.lens() == [0, 0]
