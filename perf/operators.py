"""What is measured of the packed-prompt operators: the cases, their inputs, their plain forms.

Four operators carry a batch of prompts of different lengths into the paged cache:

* ``batch_tables``: block tables and slot maps from request lengths, on the GPU;
* ``rope_append``: rotation of the packed q / k rows and the scatter of k / v by slot;
* ``prompt_attention``: causal attention over whole packed prompts with grouped heads;
* ``prompt_linear``: matrix product with bias, activation and residual in its epilogue.

``run`` computes an operator in elementary torch operations in 32 bits, or, where ``own`` is
true, makes the calls that a user makes of the package.  ``exact`` computes the same
definitions in 64 bits, written apart.
"""
import math
import random

import torch

own = False

DEV = "cuda"
DT = {"f16": torch.float16, "f32": torch.float32}


# ---- cases ------------------------------------------------------------------------------
def listed():
    return [
        # -- batch_tables
        # a decode step of 64 running sequences (contexts of 256 to 2048 in 16-token
        # blocks): one new token each, a new block now and then
        dict(name="tables_step", op="tables", seqs=64, cached_lo=256, cached_hi=2048, new_lo=1,
             new_hi=1, block=16, lens_seed=1, pad=0, assign=True),
        # admission of 512 prompts of 0 to 512 new tokens, some after cached ones
        dict(name="tables_prompts", op="tables", seqs=512, cached_lo=0, cached_hi=700, new_lo=0,
             new_hi=512, block=16, lens_seed=2, pad=37, assign=True),
        # -- rope_append
        # the tail of a chunked batch: 33 rows, 9 / 3 heads of 64
        dict(name="append_small", op="append", lens_lo=1, lens_hi=20, seqs=3, hq=9, hkv=3, d=64,
             block=16, dtype="f16", lens_seed=3, pad=2, far=False),
        # packed prompts of up to 2048 tokens, 32 / 8 heads of 128, far positions
        dict(name="append_large", op="append", lens_lo=400, lens_hi=2048, seqs=16, hq=32, hkv=8,
             d=128, block=16, dtype="f16", lens_seed=4, pad=5, far=True),
        # F32 cache, 9 / 3 heads of 64
        dict(name="append_f32", op="append", lens_lo=1, lens_hi=600, seqs=24, hq=9, hkv=3, d=64,
             block=32, dtype="f32", lens_seed=5, pad=0, far=False),
        # -- prompt_attention
        # one prompt of 32 tokens, 9 / 3 heads of 64: the smallest call, where latency counts
        dict(name="attn_small", op="attn", lens_lo=32, lens_hi=32, seqs=1, hq=9, hkv=3, d=64,
             dtype="f16", lens_seed=6, pad=0),
        # 64 prompts of 1 to 2048 tokens packed, 15 / 5 heads of 64
        dict(name="attn_ragged", op="attn", lens_lo=1, lens_hi=2048, seqs=64, hq=15, hkv=5, d=64,
             dtype="f16", lens_seed=7, pad=11),
        # one long prompt, 32 / 8 heads of 128
        dict(name="attn_long", op="attn", lens_lo=16384, lens_hi=16384, seqs=1, hq=32, hkv=8,
             d=128, dtype="f16", lens_seed=8, pad=0),
        # F32 prompts of up to 500 tokens, 9 / 3 heads of 64
        dict(name="attn_f32", op="attn", lens_lo=1, lens_hi=500, seqs=9, hq=9, hkv=3, d=64,
             dtype="f32", lens_seed=9, pad=1),
        # -- prompt_linear
        # a few rows (a short prompt): weight streaming and latency, bias and GELU
        dict(name="linear_small", op="linear", rows=33, k=768, n=2048, act="gelu", bias=True,
             residual=False, xpad=0),
        # gate / up projection of 16 prompts of 512 tokens with SwiGLU, 768 -> 2 x 2048
        dict(name="linear_swiglu", op="linear", rows=8192, k=768, n=2048, act="swiglu",
             bias=False, residual=False, xpad=0),
        # projection of the attention output at 32 heads of 128, bias and residual; an odd
        # number of rows
        dict(name="linear_large", op="linear", rows=8191, k=4096, n=4096, act="none", bias=True,
             residual=True, xpad=64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["tables", "append", "attn", "linear"])
    if op == "tables":
        seqs = _log(rng, 1, 512)
        step = rng.random() < 0.3
        hi = 1 if step else _log(rng, 1, 512)
        return dict(op=op, seqs=seqs, cached_lo=0, cached_hi=_log(rng, 1, 4000),
                    new_lo=1 if step else 0, new_hi=hi, block=rng.choice([8, 16, 24, 64]),
                    lens_seed=rng.randrange(1 << 20), pad=rng.randint(1, 40),
                    assign=rng.random() < 0.8)
    heads = [(9, 3), (15, 5), (12, 12), (32, 8), (8, 1), (5, 5), (6, 2)]
    if op == "append":
        hq, hkv = rng.choice(heads)
        d = rng.choice([32, 64, 80, 96, 128])
        hi = _log(rng, 1, 2048)
        return dict(op=op, lens_lo=rng.choice([0, 1, max(hi // 2, 1)]), lens_hi=hi,
                    seqs=_log(rng, 1, max(1, 20000 // hi // 4)), hq=hq, hkv=hkv, d=d,
                    block=rng.choice([8, 16, 24, 128]), dtype=rng.choice(["f16", "f16", "f32"]),
                    lens_seed=rng.randrange(1 << 20), pad=rng.randint(1, 9),
                    far=rng.random() < 0.5)
    if op == "attn":
        dtype = rng.choice(["f16", "f16", "f16", "f32"])
        hq, hkv = rng.choice(heads)
        d = rng.choice([32, 64, 64, 80, 96, 128, 128])
        hi = _log(rng, 1, 8192 if dtype == "f16" else 1024)
        return dict(op=op, lens_lo=rng.choice([0, 1, max(hi // 2, 1)]), lens_hi=hi,
                    seqs=_log(rng, 1, max(1, min(64, 16384 // hi))), hq=hq, hkv=hkv, d=d,
                    dtype=dtype, lens_seed=rng.randrange(1 << 20), pad=rng.randint(1, 20))
    act = rng.choice(["none", "none", "relu", "silu", "gelu", "swiglu"])
    return dict(op=op, rows=_log(rng, 1, 8192), k=8 * _log(rng, 4, 512), n=8 * _log(rng, 4, 512),
                act=act, bias=rng.random() < 0.5, residual=rng.random() < 0.5,
                xpad=rng.choice([0, 0, 8, 128]))


def _lens(case, lo, hi, salt=0):
    """Lengths of the case's requests: fixed by the case alone, log-spread for wide ranges."""
    r = random.Random(case["lens_seed"] * 1000003 + salt)
    out = []
    for _ in range(case["seqs"]):
        if hi > 10 * max(lo, 1) and r.random() < 0.5:
            out.append(max(lo, _log(r, max(lo, 1), hi)))
        else:
            out.append(r.randint(lo, hi))
    return out


# ---- inputs -----------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = random.Random(seed)

    def randn(*shape, std=1.0, dtype=torch.float16):
        return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)

    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device=DEV)

    s = dict(case=case)
    op = case["op"]
    if op == "tables":
        # lengths keep their totals over seeds (a plan of the same size), in another order
        order = list(range(case["seqs"]))
        rng.shuffle(order)
        cached = _lens(case, case["cached_lo"], case["cached_hi"])
        new = _lens(case, case["new_lo"], case["new_hi"], 1)
        cached, new = [cached[i] for i in order], [new[i] for i in order]
        bs = case["block"]
        held = [-(-c // bs) for c in cached]
        after = [-(-(c + n) // bs) for c, n in zip(cached, new)]
        mb = max(max(after), 1) + 2
        nblocks = sum(after) + 16
        ids = list(range(nblocks))
        rng.shuffle(ids)
        table = torch.full((case["seqs"], mb), -1, dtype=torch.int32)
        at = 0
        for i, (h, a) in enumerate(zip(held, after)):
            h = h if case["assign"] else a  # without assignment every block is there already
            table[i, :h] = torch.tensor(ids[at:at + h], dtype=torch.int32)
            at += h
        s.update(table=table.to(DEV), cached=ints(cached), new=ints(new), bs=bs,
                 rows=sum(new) + case["pad"], nblocks=nblocks,
                 free=ints(ids[at:]) if case["assign"] else None)
        if own:
            import rustllm_b200 as rb
            # the tables need no K/V storage: a descriptor over one-row arenas
            s["arena"] = torch.empty((nblocks, 1, bs, 2), dtype=torch.float16, device=DEV)
            s["kv"] = rb.paged_kv_from_tensors(s["arena"], s["arena"], s["table"], s["cached"])
            s["maps"] = rb.BatchTables.empty(case["seqs"], s["rows"], DEV)
    elif op == "append":
        lens = _lens(case, case["lens_lo"], case["lens_hi"])
        dt = DT[case["dtype"]]
        hq, hkv, d, bs = case["hq"], case["hkv"], case["d"], case["block"]
        t, rows = sum(lens), sum(lens) + case["pad"]
        # first positions are the case's own: they set the number of blocks
        r = random.Random(case["lens_seed"])
        first = [r.randrange(0, 120000 if case["far"] else 64) for _ in lens]
        pos = [f + i for f, n in zip(first, lens) for i in range(n)] + [-1] * case["pad"]
        # every sequence's positions in its own shuffled blocks
        held = [(f % bs + n + bs - 1) // bs if n else 0 for f, n in zip(first, lens)]
        nblocks = sum(held) + 3
        ids = list(range(nblocks))
        rng.shuffle(ids)
        slots, at = [], 0
        for f, n, h in zip(first, lens, held):
            slots += [ids[at + (f % bs + i) // bs] * bs + (f % bs + i) % bs for i in range(n)]
            at += h
        slots += [-1] * case["pad"]
        table_len = (max(pos) if pos else 0) + 2
        theta = 100000.0
        inv = theta ** (-torch.arange(d // 2, dtype=torch.float64, device=DEV) * 2 / d)
        ang = torch.arange(max(table_len, 1), dtype=torch.float64, device=DEV)[:, None] * inv
        qkv = randn(rows, (hq + 2 * hkv) * d, dtype=dt)
        s.update(qkv=qkv, pos=ints(pos), slots=ints(slots, torch.int64),
                 cos=ang.cos().float(), sin=ang.sin().float(), t=t,
                 q_out=torch.zeros(rows, hq, d, dtype=dt, device=DEV),
                 k_out=torch.zeros(rows, hkv, d, dtype=dt, device=DEV),
                 kc=randn(nblocks, hkv, bs, d, dtype=dt), vc=randn(nblocks, hkv, bs, d, dtype=dt))
        if own:
            import rustllm_b200 as rb
            s["kv"] = rb.paged_kv_from_tensors(
                s["kc"], s["vc"], torch.zeros((1, 1), dtype=torch.int32, device=DEV),
                torch.zeros(1, dtype=torch.int32, device=DEV))
    elif op == "attn":
        lens = _lens(case, case["lens_lo"], case["lens_hi"])
        dt = DT[case["dtype"]]
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        starts = [0]
        for n in lens:
            starts.append(starts[-1] + n)
        rows = starts[-1] + case["pad"]
        # q, k, v are views of one fused projection, as a decoder has them
        s.update(qkv=randn(rows, (hq + 2 * hkv) * d, dtype=dt), starts=starts,
                 q_start=ints(starts), max_rows=max(lens),
                 out=torch.zeros(rows, hq, d, dtype=dt, device=DEV),
                 lse=torch.zeros(rows, hq, device=DEV))
    else:
        m, k, n = case["rows"], case["k"], case["n"]
        wide = 2 * n if case["act"] == "swiglu" else n
        s.update(x=randn(m, k + case["xpad"])[:, :k], w=randn(k, wide, std=1 / math.sqrt(k)),
                 bias=randn(wide, std=0.3) if case["bias"] else None,
                 residual=randn(m, n) if case["residual"] else None,
                 out=torch.zeros(m, n, dtype=torch.float16, device=DEV))
    return s


def _qkv(s):
    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    rows, x = s["qkv"].shape[0], s["qkv"]
    return (x[:, :hq * d].view(rows, hq, d), x[:, hq * d:(hq + hkv) * d].view(rows, hkv, d),
            x[:, (hq + hkv) * d:].view(rows, hkv, d))


# ---- one pass ---------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _own_tables(s):
    import rustllm_b200 as rb
    t = rb.batch_tables(s["kv"], s["new"], s["rows"], free_blocks=s["free"], out=s["maps"])
    return dict(table=s["table"], q_start=t.q_start, positions=t.positions, row_seq=t.row_seq,
                slots=t.slots, info=t.info)


def _own_append(s):
    import rustllm_b200 as rb
    q, k, v = _qkv(s)
    rb.rope_append(s["kv"], q, k, v, s["pos"], s["slots"], rope=(s["cos"], s["sin"]),
                   q_out=s["q_out"], k_out=s["k_out"])
    return dict(q=s["q_out"], k=s["k_out"], k_cache=s["kc"], v_cache=s["vc"])


def _own_attn(s):
    import rustllm_b200 as rb
    q, k, v = _qkv(s)
    rb.prompt_attention(q, k, v, s["q_start"], s["max_rows"], out=s["out"], lse=s["lse"])
    return dict(out=s["out"], lse=s["lse"])


def _own_linear(s):
    import rustllm_b200 as rb
    return rb.prompt_linear(s["x"], s["w"], bias=s["bias"], activation=s["case"]["act"],
                            residual=s["residual"], out=s["out"])


def _plain_tables(s):
    bs, rows, nblocks = s["bs"], s["rows"], s["nblocks"]
    table, cached, new = s["table"].clone(), s["cached"].long(), s["new"].long().clamp(min=0)
    b, mb = table.shape
    end = torch.cumsum(new, 0)
    q_start = torch.cat([end.new_zeros(1), end])
    total = q_start[-1]
    held = (cached + bs - 1) // bs
    fits = (cached >= 0) & (cached + new <= mb * bs)
    if s["free"] is not None:
        free = s["free"].long()
        need = torch.where(fits, (cached + new + bs - 1) // bs - held, 0)
        incl = torch.cumsum(need, 0)
        placed = fits & ((need == 0) | (incl <= free.numel()))
        col = torch.arange(mb, device=DEV)[None]
        i = col - held[:, None]
        write = placed[:, None] & (i >= 0) & (i < need[:, None])
        src = (incl - need)[:, None] + i
        table = torch.where(write, free[src.clamp(0, free.numel() - 1)].int(), table)
        taken = torch.where(placed, need, 0).sum()
    else:
        placed, taken = fits, total * 0
    r = torch.arange(rows, device=DEV)
    seq = torch.searchsorted(end, r, right=True)
    live = r < total
    sq = seq.clamp(max=b - 1)
    pos = cached[sq] + r - q_start[sq]
    ok = live & placed[sq]
    blk = table[sq, (pos // bs).clamp(0, mb - 1)].long()
    slot_ok = ok & (blk >= 0) & (blk < nblocks)
    info = torch.stack([taken, total, (~placed).sum(), (total - rows).clamp(min=0)])
    return dict(table=table, q_start=q_start.int(), positions=torch.where(ok, pos, -1).int(),
                row_seq=torch.where(live, seq, -1).int(),
                slots=torch.where(slot_ok, blk * bs + pos % bs, -1), info=info.int())


def _plain_append(s):
    q, k, v = _qkv(s)
    live = s["pos"] >= 0
    p = s["pos"].long().clamp(min=0)
    c, si = s["cos"][p][:, None], s["sin"][p][:, None]

    def rotate(x):
        h = x.shape[-1] // 2
        a, b = x[..., :h].float(), x[..., h:].float()
        return torch.cat([a * c - b * si, b * c + a * si], -1).to(x.dtype)

    qr = torch.where(live[:, None, None], rotate(q), 0)
    kr = torch.where(live[:, None, None], rotate(k), 0)
    kc, vc = s["kc"].clone(), s["vc"].clone()
    bs = s["case"]["block"]
    sl = s["slots"][:s["t"]]
    kc[sl // bs, :, sl % bs] = kr[:s["t"]]
    vc[sl // bs, :, sl % bs] = v[:s["t"]]
    return dict(q=qr, k=kr, k_cache=kc, v_cache=vc)


def _plain_attn(s):
    q, k, v = _qkv(s)
    c = s["case"]
    group, scale = c["hq"] // c["hkv"], 1.0 / math.sqrt(c["d"])
    out, lse = torch.zeros_like(s["out"]), torch.zeros_like(s["lse"])
    for lo, hi in zip(s["starts"], s["starts"][1:]):
        n = hi - lo
        if n == 0:
            continue
        step = max(1, min(n, (1 << 28) // (n * c["hq"])))
        kh = k[lo:hi].float().permute(1, 2, 0)  # [Hkv, D, n]
        vh = v[lo:hi].float().transpose(0, 1)   # [Hkv, n, D]
        for r0 in range(0, n, step):
            r1 = min(n, r0 + step)
            qh = q[lo + r0:lo + r1].float().view(r1 - r0, c["hkv"], group, c["d"])
            qh = qh.permute(1, 2, 0, 3).reshape(c["hkv"], -1, c["d"])
            sc = (torch.matmul(qh, kh[:, :, :r1]) * scale).view(c["hkv"], group, r1 - r0, r1)
            hide = (torch.arange(r1, device=DEV)[None] >
                    torch.arange(r0, r1, device=DEV)[:, None])
            sc = sc.masked_fill(hide, float("-inf"))
            m = sc.amax(-1, keepdim=True)
            p = torch.exp(sc - m)
            l = p.sum(-1, keepdim=True)
            o = torch.matmul(p.view(c["hkv"], -1, r1), vh[:, :r1]).view(
                c["hkv"], group, r1 - r0, c["d"]) / l
            out[lo + r0:lo + r1] = o.permute(2, 0, 1, 3).reshape(r1 - r0, c["hq"], c["d"]).to(out.dtype)
            lse[lo + r0:lo + r1] = (m + torch.log(l))[..., 0].permute(2, 0, 1).reshape(
                r1 - r0, c["hq"])
    return dict(out=out, lse=lse)


def _plain_linear(s):
    y = torch.matmul(s["x"].float(), s["w"].float())
    if s["bias"] is not None:
        y = y + s["bias"].float()
    act = s["case"]["act"]
    if act == "swiglu":
        n = s["case"]["n"]
        gate, up = y[:, :n], y[:, n:]
        y = gate / (1 + torch.exp(-gate)) * up
    elif act == "silu":
        y = y / (1 + torch.exp(-y))
    elif act == "relu":
        y = torch.where(y > 0, y, 0)
    elif act == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.half()


_OWN = dict(tables=_own_tables, append=_own_append, attn=_own_attn, linear=_own_linear)
_PLAIN = dict(tables=_plain_tables, append=_plain_append, attn=_plain_attn, linear=_plain_linear)


# ---- what a pass cannot do without --------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "tables":
        cached = _lens(case, case["cached_lo"], case["cached_hi"])
        new = _lens(case, case["new_lo"], case["new_hi"], 1)
        bs = case["block"]
        used = sum(-(-(c + n) // bs) - c // bs for c, n in zip(cached, new) if n)
        taken = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(cached, new))
        rows, b = sum(new) + case["pad"], case["seqs"]
        # lengths and block ids in; offsets, row maps and the new table entries out
        return dict(bytes=8 * b + 4 * used + 4 * (b + 1) + 16 * rows + 16 +
                    (4 * taken if case["assign"] else 0), flops=0)
    if op == "append":
        lens = _lens(case, case["lens_lo"], case["lens_hi"])
        e = 2 if case["dtype"] == "f16" else 4
        t, hq, hkv, d = sum(lens), case["hq"], case["hkv"], case["d"]
        # q, k, v in; q, k out; k and v into the cache; positions, slots and table rows in
        # (sequences near the start share table rows: the longest run counts there)
        trows = t if case["far"] else min(t, 64 + max(lens))
        return dict(bytes=t * d * e * ((hq + 2 * hkv) + (hq + hkv) + 2 * hkv) +
                    12 * (t + case["pad"]) + trows * d * 4, flops=3 * t * d * (hq + hkv))
    if op == "attn":
        lens = _lens(case, case["lens_lo"], case["lens_hi"])
        e = 2 if case["dtype"] == "f16" else 4
        t, hq, hkv, d = sum(lens), case["hq"], case["hkv"], case["d"]
        pairs = sum(n * (n + 1) // 2 for n in lens)
        return dict(bytes=t * d * e * 2 * (hq + hkv) + 4 * t * hq + 4 * (case["seqs"] + 1),
                    flops=4 * d * hq * pairs)
    m, k, n = case["rows"], case["k"], case["n"]
    wide = 2 * n if case["act"] == "swiglu" else n
    elems = m * k + k * wide + m * n
    elems += wide if case["bias"] else 0
    elems += m * n if case["residual"] else 0
    return dict(bytes=2 * elems, flops=2 * m * k * wide)


# ---- the definitions in 64 bits -----------------------------------------------------------
def exact(case, seed):
    op = case["op"]
    if op == "tables":
        return None  # whole numbers throughout
    s = prepare(case, seed)
    if op == "append":
        rows, hq, hkv, d, bs = s["qkv"].shape[0], case["hq"], case["hkv"], case["d"], case["block"]
        x = s["qkv"].double().reshape(rows, hq + 2 * hkv, 2, d // 2)
        turn = torch.complex(s["cos"].double(), s["sin"].double())
        z = torch.complex(x[:, :hq + hkv, 0], x[:, :hq + hkv, 1])
        t = s["t"]
        rot = torch.zeros(rows, hq + hkv, d, dtype=torch.float64, device=DEV)
        z = z[:t] * turn.index_select(0, s["pos"][:t].long())[:, None]
        rot[:t] = torch.cat([z.real, z.imag], -1)
        flat = s["slots"][:t]
        caches = []
        for arena, fresh in ((s["kc"], rot[:t, hq:]),
                             (s["vc"], x[:t, hq + hkv:].reshape(t, hkv, d))):
            # by slot: [blocks * block, Hkv, D]
            c = arena.double().transpose(1, 2).reshape(-1, hkv, d).index_copy(0, flat, fresh)
            caches.append(c.view(-1, bs, hkv, d).transpose(1, 2))
        return dict(q=rot[:, :hq], k=rot[:, hq:], k_cache=caches[0], v_cache=caches[1])
    if op == "attn":
        rows, hq, hkv, d = s["qkv"].shape[0], case["hq"], case["hkv"], case["d"]
        x = s["qkv"].double().view(rows, hq + 2 * hkv, d)
        out = torch.zeros(rows, hq, d, dtype=torch.float64, device=DEV)
        lse = torch.zeros(rows, hq, dtype=torch.float64, device=DEV)
        for i, lo in enumerate(s["starts"][:-1]):
            hi = s["starts"][i + 1]
            for h in range(hq):
                kv = hq + h // (hq // hkv)
                for a in range(lo, hi, 4096):
                    b = min(hi, a + 4096)
                    logits = torch.einsum("id,jd->ij", x[a:b, h], x[lo:b, kv]) / math.sqrt(d)
                    seen = torch.ones_like(logits, dtype=torch.bool).tril(a - lo)
                    logits = torch.where(seen, logits, -math.inf)
                    z = torch.logsumexp(logits, 1)
                    out[a:b, h] = torch.exp(logits - z[:, None]) @ x[lo:b, kv + hkv]
                    lse[a:b, h] = z
        return dict(out=out, lse=lse)
    y = s["x"].double() @ s["w"].double()
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["act"] == "swiglu":
        gate, up = y.chunk(2, 1)
        y = gate * torch.sigmoid(gate) * up
    elif case["act"] == "silu":
        y = y * torch.sigmoid(y)
    elif case["act"] == "relu":
        y = y.clamp(min=0)
    elif case["act"] == "gelu":
        y = y * torch.special.ndtr(y)
    return y + s["residual"].double() if s["residual"] is not None else y
