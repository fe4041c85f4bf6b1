"""The cache in eight bits, attention of drafted tokens over it, and log probabilities of given tokens: each operator
against its formula in 64 bits, at the sizes and masks where it can go wrong.  Pages that a request does not own and cells it has
not written hold NaN.

Tolerances: a rounding to nearest is off by half a step of its type (bfloat16 2^-8, float16 2^-11, e4m3 2^-4 of the value; a code
under 2^-6 by 2^-10 of its vector's power of two).  An attention result is sum p v / sum p with p rounded once in both sums (U_P), scores off by at most
their sum's D float32 roundings, and one rounding of the result:
    |error| <= U_OUT |o| + 2 (U_P + e_s + 2^-20) sum p |v|,   e_s = (D + 8) 2^-23 max sum |q k| scale
(2^-20: exponentials and their float32 sums of up to a few thousand terms, whose roundings mostly cancel)."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn
PAGE = 64


def status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def exponent(x):
    """The definition, on float64 vectors (last axis)."""
    a = x.abs()
    amax = torch.where(torch.isfinite(a), a, torch.zeros_like(a)).amax(-1)
    m, e = torch.frexp(amax)
    e = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, e, torch.full_like(e, -60)).clamp(-60, 119)


def poison(pages, kv_heads, dim, eight):
    if eight:
        k, v = [torch.full((pages, kv_heads, PAGE, dim), 0x7F, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2)]
        return k, v, *[torch.full((pages, kv_heads, PAGE), 130, dtype=torch.uint8, device=DEV) for _ in range(2)]
    return *[torch.full((pages, kv_heads, PAGE, dim), math.nan, dtype=torch.bfloat16, device=DEV) for _ in range(2)], None, None


def values(pages, exps):
    """The numbers that pages stand for, float64."""
    if exps is None:
        return pages.double()
    return torch.ldexp(pages.view(torch.uint8).cpu().view(E4M3).double(), exps.cpu().int()[..., None] - 127).to(DEV)


def tables(contexts, spare=3, seed=0):
    rng = random.Random(seed)
    blocks = [-(-c // PAGE) for c in contexts]
    order = list(range(sum(blocks) + spare))
    rng.shuffle(order)
    width = max(blocks + [1])
    return [[order.pop() for _ in range(b)] + [-1] * (width - b) for b in blocks], sum(blocks) + spare


def frequencies(n_rot):
    exact = torch.tensor([10000.0 ** (-2.0 * i / max(n_rot, 1)) for i in range(n_rot // 2)] or [0.0], dtype=torch.float64)
    high = exact.float()
    return exact, torch.stack([high, (exact - high.double()).float()]).to(DEV)


def turned(x, positions, exact, n_rot, pairing):
    x = x.clone()
    angle = torch.tensor(positions, dtype=torch.float64)[:, None, None] * exact[:n_rot // 2]
    c, s = angle.cos(), angle.sin()
    one, two = (slice(0, n_rot // 2), slice(n_rot // 2, n_rot)) if pairing == "half" else (slice(0, n_rot, 2), slice(1, n_rot, 2))
    a, b = x[..., one].clone(), x[..., two].clone()
    x[..., one], x[..., two] = a * c - b * s, a * s + b * c
    return x


# ---- the write and the reading back ------------------------------------------------------------------------------

@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("H,G,D,n_rot,pairing,parts,bias", [
    (4, 2, 16, 16, "half", 0, False), (6, 2, 32, 32, "adjacent", 3, True), (5, 5, 48, 24, "half", 1, False), (8, 2, 64, 64, "half", 9, True),
    (3, 1, 80, 0, "half", 0, False), (4, 4, 96, 96, "adjacent", 0, False), (2, 1, 112, 2, "adjacent", 2, False), (32, 8, 128, 128, "half", 4, False),
    (2, 2, 256, 128, "half", 0, False), (7, 1, 128, 128, "adjacent", 0, False),
    (8, 2, 64, 64, "half", 0, False), (5, 2, 64, 64, "adjacent", 0, False), (17, 4, 128, 128, "half", 0, False), (32, 8, 128, 64, "half", 0, False)])
def test_store_writes_cells_and_turns_by_positions(H, G, D, n_rot, pairing, parts, bias, eight):
    from lgml_b200 import ops

    g = torch.Generator().manual_seed(D + H)
    pos0, lens = [0, 61, 1000, 63], [1, 7, 40, 2]
    N, width = sum(lens), (H + 2 * G) * D
    table, pages = tables([p + n for p, n in zip(pos0, lens)])
    seq = [s for s, n in enumerate(lens) for _ in range(n)]
    cells = [p + i for p, n in zip(pos0, lens) for i in range(n)]
    positions = [max(0, c - (c % 3)) + (131072 if s == 2 else 0) for c, s in zip(cells, seq)]
    if parts:
        data = torch.randn(parts, N, width, generator=g) * torch.exp(torch.randn(width, generator=g))
        b = torch.randn(width, generator=g) if bias else None
        full = data.double().sum(0) + (b.double() if bias else 0)
        qkv = ops.Partials(data.to(DEV), b.to(DEV) if bias else None)
    else:
        wide = (torch.randn(N, width + 24, generator=g) * torch.exp(torch.randn(width + 24, generator=g))).to(torch.bfloat16)
        full = wide[:, 8:8 + width].double()
        qkv = wide.to(DEV)[:, 8:8 + width]                       # rows apart
    # float32 roundings: the sum of the parts, the rotation
    scale_of = (data.double().abs().sum(0) if parts else full.abs()).view(N, H + 2 * G, D).amax(-1, keepdim=True)
    slack = (parts + 8) * 2.0 ** -24 * scale_of * 2
    exact, freq = frequencies(n_rot)
    x = full.view(N, H + 2 * G, D)
    turn = torch.cat([turned(x[:, :H + G], positions, exact, n_rot, pairing), x[:, H + G:]], 1)
    k, v, ke, ve = poison(pages, G, D, eight)
    before = [t.clone() for t in (k, v)]
    st = status()
    q = ops.rope_kv_store(qkv, ints(positions), ints(seq), ints(table), freq, n_rot, pairing, k, v, H, G, D, st, cells=ints(cells), k_exps=ke, v_exps=ve)
    assert st.item() == 0
    want = turn[:, :H]
    assert ((q.double().cpu().view(N, H, D) - want).abs() <= 2.0 ** -8 * want.abs() + slack[:, :H] * 1.01).all()
    page = torch.tensor([table[s][c // PAGE] for s, c in zip(seq, cells)])
    at = torch.tensor(cells) % PAGE
    written = torch.zeros(pages, PAGE, dtype=torch.bool)
    written[page, at] = True
    for pool, exps, old, lo in ((k, ke, before[0], H), (v, ve, before[1], H + G)):
        want = turn[:, lo:lo + G]
        got = values(pool, exps).cpu()[page, :, at]
        err = (got - want).abs()
        if eight:
            e = exps.cpu()[page, :, at].int() - 127
            off = slack[:, lo:lo + G, 0]
            near = exponent(want)
            lo_e, hi_e = exponent(want * (1 - 1e-5)), exponent(want * (1 + 1e-5))
            assert ((e == near) | (e == lo_e) | (e == hi_e)).all()
            step = torch.ldexp(torch.ones_like(got), e[..., None].expand_as(got))
            assert (err <= torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * step) + off[..., None] * 1.07).all()
            assert torch.equal(exps.cpu().permute(0, 2, 1)[~written], torch.full_like(exps.cpu().permute(0, 2, 1)[~written], 130))
        else:
            assert (err <= 2.0 ** -8 * want.abs() + slack[:, lo:lo + G] * 1.01).all()
        raw = lambda t: (t.view(torch.uint8) if eight else t.view(torch.int16)).cpu().permute(0, 2, 1, 3)  # noqa: E731
        assert torch.equal(raw(pool)[~written], raw(old)[~written])


@pytest.mark.parametrize("N,D,pairing", [(40, 128, "half"), (40, 96, "adjacent"), (500, 128, "half"), (500, 64, "adjacent")])
def test_keys_in_codes_are_those_of_the_rotation_in_64_bits(N, D, pairing):
    """Both kernels; positions up to 500,000.  (float32's sine alone would put a few of 10^6 codes on the other side of a border.)"""
    from lgml_b200 import ops

    H, G = 2, 8
    g = torch.Generator().manual_seed(N + D)
    qkv = torch.randn(N, (H + 2 * G) * D, generator=g).to(torch.bfloat16)
    positions = [(i * 997) % 500000 for i in range(N)]
    table, pages = tables([N])
    exact, freq = frequencies(D)
    k, v, ke, ve = poison(pages, G, D, True)
    st = status()
    ops.rope_kv_store(qkv.to(DEV), ints(positions), ints([0] * N), ints(table), freq, D, pairing, k, v, H, G, D, st, cells=ints(range(N)), k_exps=ke, v_exps=ve)
    assert st.item() == 0
    page, at = torch.tensor([table[0][c // PAGE] for c in range(N)]), torch.arange(N) % PAGE
    x = turned(qkv.double().view(N, H + 2 * G, D)[:, H:H + G], positions, freq.double().sum(0).cpu(), D, pairing).float()
    e = exponent(x.double())
    assert torch.equal(ke.cpu()[page, :, at].int(), (e + 127).int())
    assert torch.equal(k.view(torch.uint8).cpu()[page, :, at], torch.ldexp(x, -e[..., None]).to(E4M3).view(torch.uint8))


def test_store_of_special_vectors_and_back():
    """Zeros, the largest and the smallest numbers, NaN and infinities; a vector read back and written again keeps its codes."""
    from lgml_b200 import ops

    D = 64
    g = torch.Generator().manual_seed(3)
    rows = torch.randn(10, D, generator=g)
    rows[0] = 0
    rows[1] *= 1e37
    rows[1, 5] = torch.finfo(torch.bfloat16).max
    rows[2] *= 1e-30
    rows[3, 7], rows[3, 9], rows[3, 60] = math.inf, -math.inf, math.nan
    rows[4] = math.nan
    rows[5] = -0.0
    rows[6] = 448.0 * 2.0 ** torch.arange(0, -64, -1)
    rows[7] = 0
    rows[7, 63] = 1e-38
    rows[8] = math.inf
    qkv = torch.cat([torch.randn(10, D, generator=g), rows, rows.flip(1)], 1).to(torch.bfloat16)
    table, st = ints([[1]]), status()
    k, v, ke, ve = poison(3, 1, D, True)
    zero = torch.zeros(1, device=DEV)
    args = (ints(list(range(10))), ints([0] * 10), table, zero, 0, "half")
    ops.rope_kv_store(qkv.to(DEV), *args, k, v, 1, 1, D, st, k_exps=ke, v_exps=ve)
    x = qkv[:, D:2 * D].double()
    e = ke[1, 0, :10].cpu().int() - 127
    assert torch.equal(e, exponent(x).int())
    got = values(k, ke)[1, 0, :10].cpu()
    finite = torch.isfinite(x)
    assert torch.isnan(got[~finite]).all() and torch.isfinite(got[finite]).all()
    step = torch.ldexp(torch.ones(10, D, dtype=torch.float64), e[:, None].expand(10, D))
    top = 448 * step                                                # (the largest numbers stop there)
    want = torch.where(finite, x, torch.zeros_like(x)).clamp(-top, top)
    assert ((got - want).abs()[finite] <= torch.maximum(2.0 ** -4 * want.abs(), 2.0 ** -10 * step)[finite]).all()
    assert (got[6, :9] == x[6, :9]).all()
    k_back, v_back = ops.kv_read(k, v, ke, ve, ints([1]), st)
    assert torch.equal(torch.nan_to_num(k_back[0, 0, :10].double().cpu(), nan=7e30), torch.nan_to_num(got, nan=7e30))
    assert torch.equal(torch.nan_to_num(v_back[0, 0, :10].cpu()), torch.nan_to_num(k_back[0, 0, :10].cpu().flip(1)))
    again = poison(3, 1, D, True)
    ops.rope_kv_store(torch.cat([k_back[0, 0, :10]] * 3, 1).contiguous(), *args, again[0], again[1], 1, 1, D, st, k_exps=again[2], v_exps=again[3])
    code = lambda t: t.view(torch.uint8)[1, 0, :10].cpu()  # noqa: E731
    keep = finite & (x.abs().amax(-1, keepdim=True) < 1e38)         # (the largest vector's first code stopped at 448, one power lower than its neighbours)
    assert torch.equal(code(again[0])[keep], code(k)[keep])
    assert st.item() == 0


def test_store_without_a_page_or_outside_the_tables_writes_nothing():
    from lgml_b200 import ops

    D, H, G = 32, 2, 1
    x = torch.randn(5, (H + 2 * G) * D, device=DEV).to(torch.bfloat16)
    _, freq = frequencies(D)
    for eight in (True, False):
        for seq, cells, table in (([0] * 5, [64, 65, 66, 67, 68], [[0, -1]]), ([0] * 5, [0, 1, 2, 3, 4], [[9, 9]]), ([0] * 5, [-1, -5, 128, 200, 1 << 30], [[0, 0]]),
                                  ([1, 2, -1, 1, 1], [0] * 5, [[0, 0]])):
            k, v, ke, ve = poison(2, G, D, eight)
            old = [t.clone().view(torch.uint8) for t in (k, v)]
            st = status()
            q = ops.rope_kv_store(x, ints([3] * 5), ints(seq), ints(table), freq, D, "half", k, v, H, G, D, st, cells=ints(cells), k_exps=ke, v_exps=ve)
            assert st.item() == 2 and torch.isfinite(q).all()
            assert torch.equal(k.view(torch.uint8), old[0]) and torch.equal(v.view(torch.uint8), old[1])
    k, v, ke, ve = poison(2, G, D, True)
    st = status()
    ops.rope_kv_store(x, ints([3] * 5), ints([0] * 5), ints([[0]]), freq, D, "half", k, v, H, G, D, st, k_exps=ke, v_exps=ve, write_kv=False)
    assert st.item() == 0 and torch.isnan(k.float()).all()


@pytest.mark.parametrize("G,D", [(1, 16), (3, 48), (8, 128), (2, 80), (1, 256)])
def test_read_is_exact_and_leaves_what_it_is_not_given(G, D):
    from lgml_b200 import ops

    g = torch.Generator().manual_seed(D)
    pool = torch.randint(0, 256, (2, 9, G, PAGE, D), generator=g, dtype=torch.uint8).to(DEV)
    exps = torch.randint(67, 247, (2, 9, G, PAGE), generator=g, dtype=torch.uint8).to(DEV)
    which = [8, 0, -1, 3, 3, 9, 1 << 30, 2]
    outs = [torch.full((len(which), G, PAGE, D), 5.0, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    st = status()
    k, v = pool[0].view(E4M3), pool[1].view(E4M3)
    got = ops.kv_read(k, v, exps[0], exps[1], ints(which), st, *outs)
    assert st.item() == 3 and got[0] is outs[0] and got[1] is outs[1]
    for out, pages, e in ((outs[0], k, exps[0]), (outs[1], v, exps[1])):
        want = values(pages, e)
        for i, p in enumerate(which):
            expect = want[p] if 0 <= p < 9 else torch.full_like(want[0], 5.0)
            # (448 x 2^119 and the codes above 256 x 2^119 are within float32; a power of 2^119 with a code over 256 fits bfloat16 too)
            assert torch.equal(torch.nan_to_num(out[i].double(), nan=1e31), torch.nan_to_num(expect, nan=1e31))
    assert ops.kv_read(k, v, exps[0], exps[1], ints([]), st)[0].shape == (0, G, PAGE, D)


# ---- attention ----------------------------------------------------------------------------------------------------

class Problem:
    """Requests with written cells, new tokens among the last of them."""

    def __init__(self, lens, pos0, H, G, D, eight, tree=False, seed=0, sharp=2.0):
        g = torch.Generator().manual_seed(seed + D + H)
        rng = random.Random(seed)
        self.H, self.G, self.D, self.lens, self.pos0, self.scale = H, G, D, lens, pos0, 1 / math.sqrt(D)
        self.table, pages = tables([p + n for p, n in zip(pos0, lens)], seed=seed)
        self.k, self.v, self.ke, self.ve = poison(pages, G, D, eight)
        self.start = [0]
        for n in lens:
            self.start.append(self.start[-1] + n)
        self.positions, self.masks = [], []
        for s, n in enumerate(lens):
            depth, mask = [], []
            for i in range(n):
                p = rng.randrange(max(-1, i - 5), i) if tree else i - 1
                depth.append(0 if p < 0 else depth[p] + 1)
                mask.append((0 if p < 0 else mask[p]) | 1 << i)
            self.positions += [pos0[s] + d for d in depth]
            self.masks += mask
        self.tree = tree
        N = self.start[-1]
        self.q = (torch.randn(N, H * D, generator=g) * sharp).to(torch.bfloat16).to(DEV)
        for s, n in enumerate(lens):
            c = pos0[s] + n
            if c == 0:
                continue
            for pool, exps, size in ((self.k, self.ke, torch.exp(torch.randn(c, G, 1, generator=g))), (self.v, self.ve, torch.exp(2 * torch.randn(c, G, 1, generator=g)))):
                x = torch.randn(c, G, D, generator=g) * size
                page = torch.tensor([self.table[s][i // PAGE] for i in range(c)])
                at = torch.arange(c) % PAGE
                if eight:
                    e = exponent(x.double())
                    pool.view(torch.uint8)[page, :, at] = torch.ldexp(x, -e[..., None]).to(E4M3).view(torch.uint8).to(DEV)
                    exps[page, :, at] = (e + 127).to(torch.uint8).to(DEV)
                else:
                    pool[page, :, at] = x.to(torch.bfloat16).to(DEV)

    def visible(self):
        return torch.tensor([m - (1 << 64) if m >> 63 else m for m in self.masks], dtype=torch.int64, device=DEV)

    def run(self, window=0, most=None, longest=None, n_splits=None, out=None, st=None, q=None, **kw):
        from lgml_b200 import ops

        q = self.q if q is None else q
        out = torch.empty(self.q.shape, dtype=torch.bfloat16, device=DEV) if out is None else out
        own = st is None
        st = status() if own else st
        ops.tree_attention(q, ints(self.positions), ints(self.start), ints(self.pos0), ints(self.table), self.k, self.v, out, self.H, self.scale, window, st,
                           max_new_tokens=most or max(max(self.lens), 1), max_kv_len=longest or max(p + n for p, n in zip(self.pos0, self.lens)), k_exps=self.ke, v_exps=self.ve,
                           visible=self.visible() if self.tree else None, n_splits=n_splits, **kw)
        if own:
            assert st.item() == 0
        return out

    def check(self, out, window=0, skip=()):
        kv = [values(p, e).cpu() for p, e in ((self.k, self.ke), (self.v, self.ve))]
        u_p = 2.0 ** -11 if self.ke is not None else 2.0 ** -8
        scale = self.scale
        for s, n in enumerate(self.lens):
            if n == 0 or s in skip:
                continue
            c, p0, r0 = self.pos0[s] + n, self.pos0[s], self.start[s]
            page, at = torch.tensor([self.table[s][i // PAGE] for i in range(c)]), torch.arange(c) % PAGE
            k, v = kv[0][page, :, at], kv[1][page, :, at]                       # [c, G, D]
            where = torch.tensor(list(range(p0)) + self.positions[r0:r0 + n])
            sees = torch.ones(n, c, dtype=torch.bool)
            for i in range(n):
                sees[i, p0:] = torch.tensor([(self.masks[r0 + i] >> j) & 1 == 1 for j in range(n)])
                if window:
                    sees[i] &= where > self.positions[r0 + i] - window
            q = self.q[r0:r0 + n].double().cpu().view(n, self.G, self.H // self.G, self.D)
            kk = torch.where(sees.any(0)[:, None, None], k, torch.zeros_like(k))
            score = torch.einsum("ngrd,cgd->grnc", q, kk) * scale
            size = torch.einsum("ngrd,cgd->grnc", q.abs(), kk.abs()).amax() * abs(scale)
            score = score.masked_fill(~sees, -math.inf)
            top = score.amax(-1, keepdim=True)
            p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total == 0, torch.ones_like(total), total)
            pv = lambda w, x: torch.einsum("grnc,cgd->ngrd", w, x)  # noqa: E731
            bad = ~torch.isfinite(v)
            clean = torch.where(bad, torch.zeros_like(v), v)
            want, mass = pv(p, clean), pv(p, clean.abs())
            reach = lambda b: (torch.einsum("nc,cgd->ngd", sees.double(), b.double())[:, :, None] > 0).expand_as(want)  # noqa: E731
            want = torch.where(reach(v == math.inf), torch.full_like(want, math.inf), want)       # (p > 0: p x infinity, and NaN where a NaN is seen)
            want = torch.where(reach(torch.isnan(v)), torch.full_like(want, math.nan), want)
            nan = reach(bad)
            got = out[r0:r0 + n].double().cpu().view_as(want)
            # a probability under float32's smallest normal number, 2^-126, may be zero there, and zero x infinity is NaN
            strong = pv((p >= 2.0 ** -126).double(), (v == math.inf).double()) > 0
            got = torch.where((want == math.inf) & ~strong & torch.isnan(got), want, got)
            assert torch.equal(torch.nan_to_num(got[nan], nan=7.0), torch.nan_to_num(want[nan], nan=7.0)) and torch.isfinite(got[~nan]).all(), s
            bound = 2.0 ** -8 * want.abs() + 2 * (u_p + (self.D + 8) * 2.0 ** -23 * size + 2.0 ** -20) * mass + 1e-30
            ok = ((got - want).abs() <= bound) | nan
            assert ok.all(), (s, float(((got - want).abs() / bound)[~nan].max()))


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("H,G,D", [(4, 4, 16), (6, 2, 32), (5, 5, 48), (8, 1, 64), (16, 4, 80), (9, 3, 96), (4, 2, 112), (32, 8, 128), (40, 2, 128), (17, 1, 64)])
def test_attention_of_one_token_at_every_head_size(H, G, D, eight):
    p = Problem([1] * 6, [0, 1, 63, 64, 200, 777], H, G, D, eight)
    for n_splits in (None, 1, 3):
        p.check(p.run(n_splits=n_splits))


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("lens,pos0,tree", [([5, 1, 3], [0, 100, 61], False), ([64, 17], [0, 1000], False), ([64, 2, 33, 64], [130, 0, 63, 1], True), ([0, 7, 0, 1], [5, 65, 0, 64], True),
                                            ([2], [4095], True), ([31], [0], True)])
@pytest.mark.parametrize("H,G,D", [(8, 2, 64), (32, 8, 128), (6, 2, 32)])
def test_attention_of_chains_and_trees(H, G, D, lens, pos0, tree, eight):
    p = Problem(lens, pos0, H, G, D, eight, tree=tree, seed=len(lens))
    for n_splits in (None, 1, 7, 12):
        p.check(p.run(n_splits=n_splits))


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("window", [1, 3, 64, 65, 500])
def test_attention_under_a_window(window, eight):
    for tree, lens in ((False, [1, 1, 1]), (True, [20, 64, 5])):
        p = Problem(lens, [0, 300, 640], 8, 2, 64, eight, tree=tree, seed=window)
        for n_splits in (None, 4):
            p.check(p.run(window=window, n_splits=n_splits), window=window)


@pytest.mark.parametrize("eight", [True, False])
def test_attention_rows_that_see_nothing_and_hidden_values_that_are_not_finite(eight):
    """Masks without a bit, a token that does not see itself, and NaN in the values (and keys) of drafted tokens that some rows do not see."""
    lens, pos0 = [9, 30], [0, 70]
    p = Problem(lens, pos0, 8, 2, 64, eight, tree=True, seed=5)
    p.masks[0] = 0                       # nothing at all: zeros
    p.masks[4] &= ~(1 << 4)              # its parents only
    p.masks[9 + 3] = 0                   # the old cells only
    for s, j, side in ((0, 2, "v"), (1, 11, "v"), (1, 11, "k"), (1, 29, "v"), (0, 8, "k")):
        c = pos0[s] + j
        pool, exps = (p.k, p.ke) if side == "k" else (p.v, p.ve)
        spot = (p.table[s][c // PAGE], slice(None), c % PAGE)
        if side == "k":                  # a key that nobody sees may hold anything
            for r in range(lens[s]):
                p.masks[(0 if s == 0 else 9) + r] &= ~(1 << j)
        if eight:
            pool.view(torch.uint8)[spot] = 0x7F if side == "k" else torch.where(torch.arange(64, device=DEV) % 3 == 0, 0x7F, 0x30).to(torch.uint8)
            if side == "k":
                exps[spot] = 255
        else:
            pool[spot] = math.nan if side == "k" else torch.where(torch.arange(64, device=DEV) % 3 == 0, math.inf if j == 2 else math.nan, 1.0).to(torch.bfloat16)
    for n_splits in (1, 2):
        out = p.run(n_splits=n_splits)
        assert (out[0] == 0).all()
        p.check(out)


@pytest.mark.parametrize("eight", [True, False])
def test_attention_leaves_longer_requests_and_the_space_between_rows_alone(eight):
    p = Problem([3, 20, 1], [10, 5, 100], 8, 2, 64, eight)
    N = 24
    wide_q = torch.full((N, 8 * 64 + 18), math.nan, dtype=torch.bfloat16, device=DEV)
    wide_q[:, 2:2 + 512] = p.q
    wide = torch.full((N, 8 * 64 + 6), 7.0, dtype=torch.bfloat16, device=DEV)
    for n_splits in (1, 3):
        p.run(most=4, n_splits=n_splits, out=wide[:, 4:4 + 512], q=wide_q[:, 2:2 + 512])
        assert (wide[3:23] == 7.0).all() and (wide[:, :4] == 7.0).all() and (wide[:, 516:] == 7.0).all()
        p.check(wide[:, 4:4 + 512], skip=(1,))


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("D", [64, 96])
def test_attention_of_the_requests_between_two_lengths(D, eight):
    """A call for the short requests and one for the longer ones are the call for all; each leaves the others' rows alone."""
    lens = [1, 40, 2, 0, 64, 3]
    p = Problem(lens, [100, 65, 0, 9, 130, 700], 8, 2, D, eight, tree=True, seed=2)
    for n_splits in (1, 3, 10):
        out = torch.full_like(p.q, 7.0)
        p.run(most=3, n_splits=n_splits, out=out)
        assert (out[1:41] == 7.0).all() and (out[43:107] == 7.0).all()
        short = out.clone()
        p.run(n_splits=n_splits, out=out, min_new_tokens=4)
        for rows in (slice(0, 1), slice(41, 43), slice(107, 110)):
            assert torch.equal(out[rows], short[rows])
        p.check(out)


@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("D", [64, 32])
def test_cached_attention_of_many_decoded_tokens_beside_short_portions(D, window):
    from types import SimpleNamespace

    from lgml_b200 import ops

    lens, pos0 = [1] * 40 + [64] + [1] * 40 + [30, 1], [5 + 7 * i for i in range(40)] + [100] + [3 * i for i in range(40)] + [0, 1000]
    p = Problem(lens, pos0, 8, 2, D, True, seed=6)
    batch = SimpleNamespace(positions=ints(p.positions), seq_start=ints(p.start), seq_pos0=ints(pos0), seq_lens=lens, max_kv_len=1001, max_q_len=64)
    cache = SimpleNamespace(block_table=ints(p.table), k=p.k, v=p.v, k_exps=p.ke, v_exps=p.ve)
    st, out = status(), torch.empty_like(p.q)
    before = ops.launch_count()
    ops.cached_attention(p.q, batch, cache, out, p.H, p.scale, window, st)
    assert ops.launch_count() - before == 2 and st.item() == 0
    p.check(out, window=window)


def test_attention_with_a_missing_page_sets_the_status():
    p = Problem([1, 1], [100, 10], 8, 2, 64, True)
    table = [row[:] for row in p.table]
    for bad in (-1, 1 << 20):
        p.table[0][1] = bad
        st = status()
        out = p.run(st=st)
        assert st.item() == 3 and torch.isfinite(out).all()
    p.table = table
    p.check(p.run())


def test_attention_of_very_large_and_small_values_and_queries():
    """Powers of two at the ends of their range, queries beyond what float16 holds."""
    for q_size, k_size, v_size in ((1e6, 1e-6, 1e30), (1e-20, 1e20, 1e-15), (3e4, 1e-3, 1.0)):
        p = Problem([1, 12], [70, 20], 8, 2, 64, True, tree=True, sharp=q_size)
        for pool, exps, size in ((p.k, p.ke, k_size), (p.v, p.ve, v_size)):
            exps.copy_((exps.int() + round(math.log2(size))).clamp(67, 246).to(torch.uint8))
        p.check(p.run(n_splits=1))
        p.check(p.run(n_splits=3))


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("H,G,D", [(24, 2, 64), (40, 5, 128), (33, 1, 64), (8, 2, 128)])
def test_attention_of_tiles_of_many_rows(H, G, D, eight):
    """Up to 2,112 rows a KV head: tiles of 128 and of 256 rows, their last ones partly filled or empty, ranges without a page."""
    for lens, pos0, window in (([64, 11, 1], [700, 130, 64], 0), ([50, 9], [0, 1500], 0), ([64, 30], [321, 63], 100)):
        p = Problem(lens, pos0, H, G, D, eight, tree=True, seed=H)
        for n_splits in (None, 1, 5, 9):
            p.check(p.run(window=window, n_splits=n_splits), window=window)


@pytest.mark.parametrize("eight", [True, False])
def test_attention_of_many_requests_with_a_few_drafted_tokens(eight):
    p = Problem([5, 8, 3] * 25, [70, 0, 64] * 25, 8, 2, 64, eight, tree=True, seed=4)
    for n_splits in (None, 2):
        p.check(p.run(n_splits=n_splits))


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-7, 2.0])
def test_attention_with_any_scale(scale, eight):
    for lens in ([1, 3], [12, 40]):
        p = Problem(lens, [100, 60], 16, 4, 64, eight, tree=True, seed=3)
        p.scale = scale
        for n_splits in (1, 3):
            p.check(p.run(n_splits=n_splits))


@pytest.mark.parametrize("lens", [[1, 3], [12, 20], [64, 40]])
@pytest.mark.parametrize("k_apart,v_apart", [(0, 7), (22, 0), (23, 3), (5, 8), (60, 60)])
def test_attention_over_vectors_of_very_different_sizes(lens, k_apart, v_apart):
    """Vectors of a page whose powers of two lie up to so many apart, and vectors of zeros between them."""
    g = torch.Generator().manual_seed(k_apart + v_apart)
    for zeros in (False, True):
        p = Problem(lens, [300, 70], 16, 4, 128, True, tree=True, seed=k_apart)
        for pool, exps, apart in ((p.k, p.ke, k_apart), (p.v, p.ve, v_apart)):
            base = 131 if apart == k_apart else 140
            exps.copy_((base - torch.randint(0, apart + 1, exps.shape, generator=g)).to(torch.uint8).to(DEV))
            exps[..., ::9] = base
            exps[..., 4::9] = base - apart
            if zeros:
                pool.view(torch.uint8)[:, :, 5::17] = 0
                exps[:, :, 5::17] = 67
        for n_splits in (1, 3):
            p.check(p.run(n_splits=n_splits))


@pytest.mark.parametrize("eight", [True, False])
def test_attention_of_many_rows_of_which_some_see_nothing_or_what_is_not_finite(eight):
    lens, pos0 = [9, 30, 40], [0, 70, 128]
    p = Problem(lens, pos0, 16, 2, 128, eight, tree=True, seed=5)
    p.masks[0] = 0
    p.masks[4] &= ~(1 << 4)
    p.masks[9 + 3] = 0
    for j in (0, 17, 39):
        p.masks[39 + j] = 0
    for s, j in ((0, 2), (1, 11), (1, 29), (2, 5)):
        c = pos0[s] + j
        spot = (p.table[s][c // PAGE], slice(None), c % PAGE)
        if eight:
            p.v.view(torch.uint8)[spot[0], :, spot[2], 3::7] = 0x7f
        else:
            p.v[spot[0], :, spot[2], 3::7] = math.nan
    old = (p.table[2][1], slice(None), 9)                  # an old cell, which all that see the old cells see
    if eight:
        p.v.view(torch.uint8)[old[0], :, old[2], 100] = 0xff
    else:
        p.v[old[0], :, old[2], 100] = math.inf
    for n_splits in (1, 2, 12):
        p.check(p.run(n_splits=n_splits))


# ---- log probabilities ----------------------------------------------------------------------------------------------

def check_logprobs(x, ids, top, got):
    x64 = x.double().cpu()
    n, v = x.shape
    logs = torch.log_softmax(x64, -1)
    plain = torch.where(torch.isnan(x64), torch.full_like(x64, -math.inf), x64)
    order = torch.argsort(plain, dim=-1, descending=True, stable=True)
    p = logs.exp()
    entropy = -torch.where(p == 0, torch.zeros_like(p), p * logs).sum(-1)
    # the float32 sums of n terms in trees of 32 to 500; logits themselves are exact; the result's own rounding
    tol = lambda want: 2e-6 + 2.0 ** -22 * want.abs()  # noqa: E731
    lp, rank, ent, top_ids, top_lp = [t.cpu() for t in got]
    assert tuple(top_ids.shape) == (n, top) and tuple(top_lp.shape) == (n, top)
    for r in range(n):
        i = int(ids[r])
        if 0 <= i < v:
            want = logs[r, i]
            assert (torch.isnan(lp[r]) and torch.isnan(want)) or lp[r] == want or abs(lp[r] - want) <= tol(want) + 2.0 ** -22 * min(abs(x64[r, i]), 1e30), (r, lp[r], want)
            if not torch.isnan(x64[r, i]):
                assert int(rank[r]) == int((order[r] == i).nonzero()[0, 0]) or torch.isnan(x64[r]).any()
        else:
            assert torch.isnan(lp[r]) and int(rank[r]) == -1
        assert (torch.isnan(ent[r]) and torch.isnan(entropy[r])) or abs(ent[r] - entropy[r]) <= 2e-6 * (1 + entropy[r].abs()), (r, ent[r], entropy[r])
        assert torch.equal(top_ids[r].long(), order[r, :top])
        for j in range(top):
            want = logs[r, order[r, j]]
            assert (torch.isnan(top_lp[r, j]) and torch.isnan(want)) or top_lp[r, j] == want or abs(top_lp[r, j] - want) <= tol(want) + 2.0 ** -22 * min(abs(x64[r, order[r, j]]), 1e30)


@pytest.mark.parametrize("n,v,top", [(1, 1, 1), (1, 1, 0), (3, 5, 5), (7, 331, 20), (2, 4096, 1), (5, 8192, 32), (3, 8193, 31), (2, 50257, 5), (1, 128256, 20), (9, 128256, 0), (700, 1000, 7),
                                     (300, 20000, 3), (1, 600000, 32)])
def test_logprobs_against_64_bits(n, v, top):
    from lgml_b200 import ops

    g = torch.Generator().manual_seed(v + n)
    wide = torch.randn(n, v + 5, generator=g) * 3
    for x in (wide.to(DEV)[:, 1:1 + v], wide[:, :v].contiguous().to(DEV)):           # rows apart and off 16 bytes, and not
        ids = torch.randint(0, v, (n,), generator=g).to(torch.int32).to(DEV)
        ids[-1] = int(x[-1].argmax())
        st = status()
        check_logprobs(x, ids, top, ops.token_logprobs(x, ids, top, st))
        assert st.item() == 0


@pytest.mark.parametrize("v", [700, 20000, 128256])
def test_logprobs_of_rows_that_are_hard(v):
    """Rising and falling logits (every entry is the best so far), equal ones, a few values, masks of -inf and of the lowest number, NaN, infinities, far from zero."""
    from lgml_b200 import ops

    g = torch.Generator().manual_seed(1)
    low = torch.finfo(torch.float32).min
    rows = [torch.arange(v) * 1e-3, -torch.arange(v) * 1e-3, torch.zeros(v), torch.randint(0, 3, (v,), generator=g).float(), torch.randn(v, generator=g) + 3e4]
    for fill in (-math.inf, low):
        masked = torch.full((v,), fill)
        masked[torch.randperm(v, generator=g)[:10]] = torch.randn(10, generator=g)
        last = torch.full((v,), fill)
        last[-1] = 2.0
        rows += [masked, last]
    rows += [torch.full((v,), low), torch.full((v,), -math.inf), torch.where(torch.arange(v) % 2 == 0, 0.0, -0.0)]
    bad = torch.randn(v, generator=g)
    bad[v // 2] = math.nan
    inf = torch.randn(v, generator=g)
    inf[3] = math.inf
    rows += [bad, inf, torch.full((v,), math.nan)]
    x = torch.stack(rows).to(DEV)
    ids = torch.randint(0, v, (len(rows),), generator=g).to(torch.int32).to(DEV)
    ids[6] = v - 1
    for top in (1, 20, 32):
        st = status()
        check_logprobs(x, ids, top, ops.token_logprobs(x, ids, top, st))
        assert st.item() == 0


def test_ranks_among_equal_logits_of_rows_off_16_bytes():
    """Ids whose logit is -inf, or one of many equal ones, in rows that start at every place of 16 bytes: in the first chunk, a later one, the last."""
    from lgml_b200 import ops

    for v in (4, 4096, 9000):
        for fill in (-math.inf, 0.0):
            wide = torch.full((8, v + 1), fill)
            wide[:, v // 2] = 1.0
            x = wide.to(DEV)[:, 1:]                      # (v + 1 odd: rows start 1, 2, 3 .. places off)
            for id in (0, 3, v - 2, v - 1):
                st = status()
                got = ops.token_logprobs(x, ints([id] * 8), 2, st)
                row = wide[0, 1:]
                want = int((row > row[id]).sum() + (row[:id] == row[id]).sum())
                assert got.ranks.tolist() == [want] * 8 and st.item() == 0, (v, fill, id)


def test_logprobs_without_an_id_and_with_one_outside():
    from lgml_b200 import ops

    x = torch.randn(4, 1000, device=DEV)
    st = status()
    check_logprobs(x, [-1, 5, -1, 999], 3, ops.token_logprobs(x, ints([-1, 5, -1, 999]), 3, st))
    assert st.item() == 0
    check_logprobs(x, [1000, 5, -2, 7], 3, ops.token_logprobs(x, ints([1000, 5, -2, 7]), 3, st))
    assert st.item() == 1
    empty = ops.token_logprobs(x[:0], ints([]), 3, st)
    assert [tuple(t.shape) for t in empty] == [(0,), (0,), (0,), (0, 3), (0, 3)]


# ---- together ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("eight", [True, False])
def test_write_attend_and_score_together_captured_and_on_another_stream(eight):
    """A step of drafted tokens as it would be used: written, attended to, scored; eagerly, and as a replayed graph whose inputs change, beside a second
    graph captured from the same buffers, on a stream of its own.  The graphs' results are the eager ones, bit for bit."""
    from lgml_b200 import ops

    H, G, D, V = 8, 2, 64, 1000
    p = Problem([12, 5], [100, 70], H, G, D, eight, tree=True, seed=9)
    N = 17
    _, freq = frequencies(D)
    head = torch.randn(H * D, V, device=DEV) * 0.1
    qkv = torch.randn(N, (H + 2 * G) * D, device=DEV).to(torch.bfloat16)
    cells = ints([100 + i for i in range(12)] + [70 + i for i in range(5)])
    seq, st, ids = ints([0] * 12 + [1] * 5), status(), ints(list(range(N)))
    pos, start, pos0, table, vis = ints(p.positions), ints(p.start), ints(p.pos0), ints(p.table), p.visible()

    def step(n_splits):
        q = ops.rope_kv_store(qkv, pos, seq, table, freq, D, "half", p.k, p.v, H, G, D, st, cells=cells, k_exps=p.ke, v_exps=p.ve)
        out = torch.empty(N, H * D, dtype=torch.bfloat16, device=DEV)
        ops.tree_attention(q, pos, start, pos0, table, p.k, p.v, out, H, 0.125, 0, st, 12, 112, k_exps=p.ke, v_exps=p.ve, visible=vis, n_splits=n_splits)
        return [q, out, *ops.token_logprobs(out.float() @ head, ids, 4, st)]

    def eager(n_splits):
        got = [t.clone() for t in step(n_splits)]
        p.q = got[0]
        p.check(got[1])
        return got

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        step(1), step(3)
    torch.cuda.synchronize()
    for n_splits in (1, 3):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs = step(n_splits)
        graphs.append((n_splits, g, outs))
    for turn in range(3):
        qkv.copy_(torch.randn_like(qkv))
        for n_splits, g, outs in graphs[::-1] if turn % 2 else graphs:
            want = eager(n_splits)
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                g.replay()
            torch.cuda.synchronize()
            for a, b in zip(outs, want):
                assert torch.equal(a, b)
    assert st.item() == 0


def test_refusals():
    from lgml_b200 import ops

    p = Problem([1, 2], [3, 9], 8, 2, 64, True)
    x = torch.randn(3, 12 * 64, device=DEV).to(torch.bfloat16)
    _, freq = frequencies(64)
    st = status()
    store = lambda **kw: ops.rope_kv_store(kw.pop("x", x), kw.pop("pos", ints([3, 9, 10])), ints([0, 1, 1]), kw.pop("table", ints(p.table)), kw.pop("freq", freq), kw.pop("n_rot", 64),  # noqa: E731
                                           kw.pop("pairing", "half"), kw.pop("k", p.k), kw.pop("v", p.v), 8, 2, 64, st, **{"k_exps": p.ke, "v_exps": p.ve, **kw})
    bf = torch.zeros_like(p.k, dtype=torch.bfloat16)
    for kw in (dict(x=x.float()), dict(x=x[:, :-64]), dict(pos=ints([1])), dict(pos=torch.zeros(3, dtype=torch.int64, device=DEV)), dict(n_rot=63), dict(n_rot=66), dict(n_rot=-2),
               dict(pairing="other"), dict(k=bf), dict(v=p.v[:, :, :, :32]), dict(k_exps=None), dict(k_exps=p.ke[:, :, :32]), dict(k_exps=p.ke.int()), dict(freq=freq[:, :8].contiguous()),
               dict(table=ints(p.table).cpu()), dict(cells=ints([1, 2])), dict(q_out=torch.zeros(3, 512, device=DEV))):
        with pytest.raises(ops.KernelError):
            store(**kw)
    for kw in (dict(most=65), dict(q=p.q[:, :-64]), dict(q=p.q.float()), dict(n_splits=257), dict(n_splits=0), dict(n_splits=9, scratch=torch.zeros(8, device=DEV)),
               dict(out=torch.zeros(3, 512, device=DEV))):
        with pytest.raises(ops.KernelError):
            p.run(**kw)
    with pytest.raises(ops.KernelError):
        ops.kv_read(bf, bf, None, None, ints([0]), st)
    for kw in (dict(top=33), dict(top=-1), dict(x=torch.zeros(2, 9, device=DEV, dtype=torch.bfloat16)), dict(x=torch.zeros(9, 2, device=DEV).t()), dict(ids=ints([1])), dict(x=torch.zeros(2, 9))):
        with pytest.raises(ops.KernelError):
            ops.token_logprobs(kw.get("x", torch.zeros(2, 9, device=DEV)), kw.get("ids", ints([1, 2])), kw.get("top", 3), st)
    assert st.item() == 0
