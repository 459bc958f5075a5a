"""The block-scaled E4M3 cache: batch tables, writes, decode and chunk attention
against plain forms in 64 bits written here from the definitions.

Whole numbers, bytes and scales have to be equal. Attention's outputs may be off by

- their own rounding, 2^-8 of the value (bf16);
- scores: D products summed in fp32, (D + 2) 2^-24 of the largest sum M of their sizes
  (scaled), which moves a weight by that factor above and the denominator below it, and
  2^-22 of the exponential: twice ((D + 2) 2^-24 M + 2^-22);
- the sums over L keys and their splits in fp32: (L + 64) 2^-24;
- chunks: weights rounded to bf16 ahead of their product, 2^-8;

all but the first of the sum of the weighted values' sizes; and weights below 2^-126 of
the largest may be lost (fp32's normal range), L 2^-126 of the largest value.
"""

import math

import pytest
import torch

from kserve_amd import ops

PAGE = 16
E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu


def devices():
    return ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def byte_values():
    """What the 256 E4M3 bytes stand for, in 64 bits."""
    v = []
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        x = (8 + m) * 2.0 ** (e - 10) if e else m * 2.0**-9
        v.append(math.nan if b & 127 == 127 else -x if b & 128 else x)
    return torch.tensor(v, dtype=torch.float64)


VALUES = byte_values()


def nearest_bytes(x):
    """E4M3 bytes nearest to x (64 bits; NaN stays, larger ones become 448), ties to the
    even byte: by distance to all of them."""
    x = x.double()
    size = x.abs().clamp(max=448.0).reshape(-1)
    pos = VALUES[:127]
    hi = torch.searchsorted(pos, size).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = size - pos[lo], pos[hi] - size
    pick = torch.where(dl < dh, lo, torch.where(dh < dl, hi, torch.where(lo % 2 == 0, lo, hi)))
    pick = torch.where(x.reshape(-1).isnan(), 127, pick)
    return (pick + 128 * torch.signbit(x).reshape(-1)).view(x.shape).to(torch.uint8)


def held(cache, scale):
    """A cache's values in 64 bits."""
    e = scale.view(torch.uint8).cpu().double() - 127
    return VALUES[cache.view(torch.uint8).cpu().long()] * torch.exp2(e)[..., None, None]


def written(x, cache, scale, slots):
    """(bytes, exponent bytes) after the rows x are written: the definition, page by page."""
    codes, exps = cache.view(torch.uint8).cpu().clone(), scale.view(torch.uint8).cpu().clone()
    block = cache.shape[2]
    pages = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < cache.shape[0] * block:
            pages.setdefault(s // block, {})[s % block] = x[t].cpu().double()
    for page, rows in pages.items():
        for h in range(cache.shape[1]):
            new = torch.stack([r[h] for r in rows.values()])
            top = float(new[new.isfinite()].abs().max()) if new.isfinite().any() else 0.0
            e = -100
            while top > 448 * 2.0**e:
                e += 1
            now = e + 127
            if 0 not in rows:
                old = int(exps[page, h])
                now = max(now, 0 if old == 255 else old)
                factor = 0.0 if old == 255 else 2.0 ** (old - now)
                if now != old:
                    codes[page, h] = nearest_bytes(VALUES[codes[page, h].long()] * factor)
            for o, r in rows.items():
                codes[page, h, o] = nearest_bytes(r[h] * 2.0 ** (127 - now))
            exps[page, h] = now
    return codes, exps


def same_bytes(got, want):
    """Equal, any not-a-number for another."""
    got = got.view(torch.uint8).cpu()
    nan = (got & 127) == 127
    assert torch.equal(nan, (want & 127) == 127)
    # zeros keep their sign
    assert torch.equal(got[~nan], want[~nan])


def make_cache(pages, kv, D, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (pages, kv, PAGE, D), generator=g, dtype=torch.int32)
    codes = torch.where(codes % 128 == 127, 0, codes).to(torch.uint8)
    exps = (118 + spread * torch.randn((pages, kv), generator=g)).round().clamp(90, 140)
    return codes.view(E4M3), exps.to(torch.uint8).view(E8M0)


class TestWrite:
    def check(self, dev, k, v, kc, vc, ks, vs, slots):
        want = [written(x, c, s, slots) for x, c, s in ((k, kc, ks), (v, vc, vs))]
        dv = [t.to(dev) for t in (kc, vc)] + [t.view(torch.uint8).to(dev).view(E8M0) for t in (ks, vs)]
        ops.reshape_and_cache(
            k if k.device.type == dev else k.to(dev), v if v.device.type == dev else v.to(dev),
            dv[0], dv[1], slots.to(dev), k_scale=dv[2], v_scale=dv[3],
        )
        for i in range(2):
            same_bytes(dv[i], want[i][0])
            assert torch.equal(dv[2 + i].view(torch.uint8).cpu(), want[i][1])
        return dv

    def rows(self, T, kv, D, seed, dev, pad=0):
        """k and v as views into wider rows (pad more elements a row)."""
        g = torch.Generator().manual_seed(seed)
        qkv = torch.randn((T, 4 * kv * D + pad), generator=g)
        qkv *= torch.exp(2 * torch.randn((T, 1), generator=g))
        qkv = qkv.to(torch.bfloat16).to(dev)
        k = qkv[:, kv * D : 2 * kv * D].view(T, kv, D) if pad == 0 else torch.as_strided(
            qkv, (T, kv, D), (qkv.stride(0), D, 1), kv * D + pad % 8
        )
        v = torch.as_strided(qkv, (T, kv, D), (qkv.stride(0), D, 1), 2 * kv * D + pad % 8)
        return k, v

    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("kv, D", [(1, 64), (8, 128), (3, 128), (9, 64)])
    @pytest.mark.parametrize("T, first, pad", [(1, 0, 0), (1, 5, 0), (37, 0, 8), (16, 16, 3), (50, 9, 1)])
    def test_runs_of_slots(self, dev, kv, D, T, first, pad):
        """Tokens of one sequence, aligned and not, whole and part pages."""
        kc, ks = make_cache(7, kv, D, 1)
        vc, vs = make_cache(7, kv, D, 2)
        k, v = self.rows(T, kv, D, 3, dev, pad)
        table = torch.tensor([4, 1, 6, 2])
        pos = torch.arange(first, first + T)
        slots = (table[pos // PAGE] * PAGE + pos % PAGE).int()
        self.check(dev, k, v, kc, vc, ks, vs, slots)

    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("T", [3, 100, 1500])
    def test_any_order(self, dev, T):
        """Slots in any order, some twice, some out of range: the page's rows are found
        wherever they stand, and the later of two rows stays."""
        g = torch.Generator().manual_seed(T)
        kc, ks = make_cache(40, 2, 64, 4)
        vc, vs = make_cache(40, 2, 64, 5)
        k, v = self.rows(T, 2, 64, 6, dev)
        slots = torch.randint(-20, 40 * PAGE + 20, (T,), generator=g, dtype=torch.int32)
        if T == 3:
            slots = torch.tensor([85, 40, 85], dtype=torch.int32)
        self.check(dev, k, v, kc, vc, ks, vs, slots)

    @pytest.mark.parametrize("dev", devices())
    def test_unusual_values(self, dev):
        """Infinities, not-a-numbers, zeros, the type's extremes and its subnormals."""
        inf, nan = math.inf, math.nan
        kc, ks = make_cache(12, 1, 64, 7)
        ks.view(torch.uint8)[3:6] = 255  # pages that hold nothing yet
        ks.view(torch.uint8)[6:9] = 0
        special = [
            [0.0], [inf], [-inf, 1.0], [nan, 2.0], [nan], [3.3895e38], [448.0, 449.0], [450.0],
            [1e-30, 1e-38], [9.2e-41], [2.0**-100 * 448], [2.0**-101 * 448, inf],
        ]
        k = torch.stack([torch.tensor((s * 64)[:64]) for s in special])
        k = k.to(torch.bfloat16).view(12, 1, 64)
        for off in (0, 7):
            slots = torch.arange(12, dtype=torch.int32) * PAGE + off
            self.check(dev, k, -k, kc, kc.clone(), ks, ks.clone(), slots)

    @pytest.mark.parametrize("dev", devices())
    def test_growing_page(self, dev):
        """A page filled token by token, each larger than the one before, holds what a
        page written at once holds, but for numbers that become subnormal on the way."""
        g = torch.Generator().manual_seed(11)
        k = torch.randn((PAGE, 2, 64), generator=g) * torch.exp2(torch.arange(16) / 4)[:, None, None]
        k = (k.sign() * k.abs().clamp(min=0.25)).to(torch.bfloat16).to(dev)
        one, two = [[t.to(dev) for t in make_cache(3, 2, 64, 8)] for _ in range(2)]
        spare = [t.clone() for t in one]
        ops.reshape_and_cache(k, k, one[0], spare[0], torch.arange(32, 48, dtype=torch.int32, device=dev),
                              k_scale=one[1], v_scale=spare[1])
        for i in range(PAGE):
            ops.reshape_and_cache(k[i : i + 1], k[i : i + 1], two[0], spare[0],
                                  torch.tensor([32 + i], dtype=torch.int32, device=dev),
                                  k_scale=two[1], v_scale=spare[1])
        assert torch.equal(one[1].view(torch.uint8), two[1].view(torch.uint8))
        assert torch.equal(one[0].view(torch.uint8), two[0].view(torch.uint8))
        assert torch.equal(two[0].view(torch.uint8), spare[0].view(torch.uint8))

    @pytest.mark.gpu
    def test_repeats_bitwise(self):
        """The same call twice leaves the same bytes."""
        k, v = self.rows(300, 4, 128, 12, "cuda")
        g = torch.Generator().manual_seed(13)
        slots = torch.randperm(64 * PAGE, generator=g)[:300].int()
        outs = []
        for _ in range(2):
            kc, ks = make_cache(64, 4, 128, 14)
            vc, vs = make_cache(64, 4, 128, 15)
            outs.append(self.check("cuda", k, v, kc, vc, ks, vs, slots))
        for a, b in zip(*outs):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def attention_case(lens, new, heads, kv, D, seed, window=0, spread=3.0):
    """A cache whose pages stand in any order, with bytes that are not numbers behind
    every context; queries for the last `new` tokens of each."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // PAGE) for n in lens]
    pages = sum(counts) + 1
    kc, ks = make_cache(pages, kv, D, seed + 1, spread)
    vc, vs = make_cache(pages, kv, D, seed + 2, spread)
    ids = torch.randperm(pages - 1, generator=g) + 1
    width = max(counts + [1]) + 1
    table = torch.zeros((len(lens), width), dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = ids[at : at + c]
        at += c
        if lens[i] % PAGE:
            for cache in (kc, vc):
                cache.view(torch.uint8)[table[i, c - 1], :, lens[i] % PAGE :] = 0x7F
    T = sum(new)
    q = (4 * torch.randn((T, heads, D), generator=g)).to(torch.bfloat16)
    cu = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
    return dict(
        q=q, kc=kc, vc=vc, ks=ks, vs=vs, table=table, cu=cu,
        ctx=torch.tensor(lens, dtype=torch.int32), window=window, scale=D**-0.5,
    )


def attention_oracle(c):
    """(outputs, what they may be off by without a rounding of the weights, sums of the
    weighted values' sizes), in 64 bits."""
    q = c["q"].double()
    T, H, D = q.shape
    k, v = held(c["kc"], c["ks"]), held(c["vc"], c["vs"])
    kv = k.shape[1]
    out, off, size = (torch.zeros((T, H, D), dtype=torch.float64) for _ in range(3))
    for i, L in enumerate(c["ctx"].tolist()):
        a, b = int(c["cu"][i]), int(c["cu"][i + 1])
        if a == b or L == 0:
            continue
        rows = c["table"][i, : -(-L // PAGE)].long()
        pos = torch.arange(L - (b - a), L)
        key = torch.arange(L)
        hid = key > pos[:, None]
        if c["window"]:
            hid |= key <= pos[:, None] - c["window"]
        for h in range(H):
            kk = k[rows, h // (H // kv)].reshape(-1, D)[:L]
            vv = v[rows, h // (H // kv)].reshape(-1, D)[:L]
            s = (q[a:b, h] @ kk.T) * c["scale"]
            M = ((q[a:b, h].abs() @ kk.abs().T) * abs(c["scale"])).masked_fill(hid, 0).amax(1)
            w = torch.softmax(s.masked_fill(hid, -math.inf), dim=1)
            w = torch.where(hid.all(1, keepdim=True), 0.0, w)
            out[a:b, h], size[a:b, h] = w @ vv, w @ vv.abs()
            rel = 2 * ((D + 2) * 2.0**-24 * M + 2.0**-22) + (L + 64) * 2.0**-24
            off[a:b, h] = rel[:, None] * size[a:b, h] + L * 2.0**-126 * vv.abs().max()
    return out, off + 2.0**-8 * out.abs(), size


def on(c, dev):
    return {n: t.view(torch.uint8).to(dev).view(t.dtype) if torch.is_tensor(t) and t.dtype in (E4M3, E8M0)
            else t.to(dev) if torch.is_tensor(t) else t for n, t in c.items()}


def decode(c, **more):
    return ops.paged_attention_decode(
        c["q"], c["kc"], c["vc"], c["table"], c["ctx"], c["scale"], window=c["window"],
        k_scale=c["ks"], v_scale=c["vs"], **more,
    )


def context(c, longest=None):
    n = longest or int((c["cu"][1:] - c["cu"][:-1]).max())
    return ops.context_attention_varlen(
        c["q"], c["kc"], c["vc"], c["table"], c["cu"], c["ctx"], n, c["scale"],
        window=c["window"], k_scale=c["ks"], v_scale=c["vs"],
    )


def near(got, c, chunk=False):
    out, off, size = attention_oracle(c)
    if chunk:
        off = off + 2.0**-8 * size
    assert got.dtype == torch.bfloat16
    far = (got.double().cpu() - out).abs() - off
    assert not got.isnan().any() and float(far.max()) <= 0, float(far.max())


class TestDecode:
    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("D", [64, 128])
    @pytest.mark.parametrize("heads, kv", [(1, 1), (8, 8), (6, 3), (12, 4), (8, 2), (5, 1), (12, 2), (14, 2), (64, 8)])
    def test_groups(self, dev, D, heads, kv):
        c = attention_case([1, 16, 17, 33, 95, 160], [1] * 6, heads, kv, D, 20)
        near(decode(on(c, dev)), c)

    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("window", [1, 15, 16, 40, 1000])
    def test_windows(self, dev, window):
        c = attention_case([1, 16, 31, 48, 300], [1] * 5, 8, 2, 64, 30, window)
        near(decode(on(c, dev)), c)

    @pytest.mark.gpu
    @pytest.mark.parametrize("D", [64, 128])
    @pytest.mark.parametrize(
        "lens, heads, kv",
        [([5000], 8, 1), ([2047, 1, 640], 16, 2), ([100 + 7 * i for i in range(40)], 32, 8),
         ([17] * 300, 8, 8), ([30] * 520, 4, 4), ([600] * 70, 8, 8)],
    )
    def test_splits_and_waves(self, D, lens, heads, kv):
        """Contexts in one part and in several, blocks of four and of eight waves."""
        c = attention_case(lens, [1] * len(lens), heads, kv, D, 40)
        near(decode(on(c, "cuda")), c)

    @pytest.mark.gpu
    @pytest.mark.parametrize("window", [0, 600])
    @pytest.mark.parametrize(
        "S, longest",
        [(64, 511), (64, 512), (65, 900), (200, 700), (256, 4000), (257, 700), (330, 600)],
    )
    def test_sequences_of_many_lengths(self, S, longest, window):
        """Long sequences among short, equal and empty ones, whichever goes first."""
        g = torch.Generator().manual_seed(S)
        lens = torch.randint(0, 200, (S,), generator=g)
        at = torch.randperm(S, generator=g)[: max(3, 8000 // longest)]
        lens[at] = torch.randint(longest // 2, longest + 1, (len(at),), generator=g)
        lens[at[0]], lens[at[1]], lens[0], lens[S - 1] = longest, longest, 0, longest - 1
        c = attention_case(lens.tolist(), [1] * S, 8, 8, 64, 45, window)
        near(decode(on(c, "cuda")), c)

    @pytest.mark.gpu
    @pytest.mark.parametrize(
        "S, long, heads, kv, D, window",
        [(32, [8192], 8, 8, 64, 0), (40, [40000, 9000], 16, 8, 64, 0), (64, [12000], 8, 8, 128, 0),
         (200, [4097, 8300], 8, 4, 64, 0), (256, [9000] * 30, 4, 4, 64, 0), (256, [8191, 100000], 4, 2, 64, 0),
         (1, [70000], 8, 8, 64, 0), (4, [70000, 8200], 8, 8, 64, 0), (15, [33000], 8, 8, 128, 0),
         (20, [9000, 30000], 16, 8, 64, 0), (22, [9000], 8, 8, 64, 0), (7, [30000], 8, 8, 64, 9000),
         (257, [9000], 2, 2, 64, 0), (70, [20000, 30000], 64, 8, 64, 8200), (64, [9000] * 64, 8, 8, 64, 0)],
    )
    def test_long_sequences_among_short(self, S, long, heads, kv, D, window):
        """Some so long that other blocks take parts of them, as many as there are."""
        g = torch.Generator().manual_seed(S)
        lens = torch.randint(0, 120, (S,), generator=g)
        lens[torch.randperm(S, generator=g)[: len(long)]] = torch.tensor(long)
        c = attention_case(lens.tolist(), [1] * S, heads, kv, D, 46, window)
        d = on(c, "cuda")
        got = decode(d)
        near(got, c)
        assert torch.equal(got, decode(d))

    @pytest.mark.gpu
    @pytest.mark.parametrize("S", [12, 40, 70])
    def test_replayed_with_other_lengths(self, S):
        """A captured call whose long sequences are others at every replay."""
        g = torch.Generator().manual_seed(S)
        c = attention_case([8992] + [16] * (S - 1), [1] * S, 16, 8, 64, 47)
        ids = c["table"][0, :562]
        c["table"] = torch.stack([ids[torch.randperm(562, generator=g)] for _ in range(S)])
        d = on(c, "cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            decode(d)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = decode(d)
        for long in ([], [0], [S - 1, 3], [1, 2, 5, 6, 7, 8], list(range(S))):
            c["ctx"] = torch.randint(0, 90, (S,), generator=g).int()
            c["ctx"][long] = torch.randint(4000, 8993, (len(long),), generator=g).int()
            d["ctx"].copy_(c["ctx"])
            graph.replay()
            near(got, c)
            assert torch.equal(got, decode(d))

    @pytest.mark.parametrize("dev", devices())
    def test_extreme_scales(self, dev):
        """Pages from 2^-90 to 2^13 beside one another."""
        c = attention_case([100, 64], [1, 1], 4, 2, 128, 50)
        c["ks"].view(torch.uint8)[::3] = 37
        c["vs"].view(torch.uint8)[::2] = 140
        near(decode(on(c, dev)), c)

    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("empty", [0, -3])
    def test_empty_context_and_out(self, dev, empty):
        """A sequence without keys gives zeros; `out` is filled and returned."""
        c = attention_case([40, 1, 20], [1] * 3, 8, 2, 128, 60)
        c["ctx"][1] = empty
        d = on(c, dev)
        out = torch.full_like(d["q"], 7.0)
        assert decode(d, out=out) is out
        assert not out[1].any()
        c["ctx"][1] = 0
        near(out, c)

    @pytest.mark.parametrize("dev", devices())
    def test_tables_without_columns(self, dev):
        """Nothing to read: zeros, whatever the lengths say."""
        c = attention_case([40, 30], [1, 1], 8, 2, 64, 65)
        d = on(c, dev)
        d["table"] = d["table"][:, :0].contiguous()
        assert not decode(d).any()
        assert not context(d).any()
        assert not context(d, 40).any()

    @pytest.mark.gpu
    def test_strided_queries_and_negative_scale(self):
        c = attention_case([40, 100], [1] * 2, 8, 2, 64, 70)
        c["scale"] = -c["scale"]
        d = on(c, "cuda")
        wide = torch.zeros((2, 12, 64), dtype=torch.bfloat16, device="cuda")
        wide[:, 2:10] = d["q"]
        d["q"] = wide[:, 2:10]
        near(decode(d), c)

    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("window", [0, 30])
    def test_ids_outside_the_cache(self, dev, window):
        """Table entries and lengths out of range stay inside the cache."""
        c = attention_case([40, 100], [1] * 2, 8, 2, 128, 80, window)
        d = on(c, dev)
        d["table"][0, 1], d["table"][0, 2] = -5, 1 << 30
        d["ctx"][0] = 1 << 30
        got = decode(d)
        c["q"], c["cu"], c["ctx"], c["table"] = c["q"][1:], c["cu"][:2], c["ctx"][1:], c["table"][1:]
        near(got[1:], c)


class TestContext:
    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("D", [64, 128])
    @pytest.mark.parametrize("heads, kv", [(1, 1), (6, 2), (8, 2), (7, 1)])
    def test_chunks(self, dev, D, heads, kv):
        c = attention_case([1, 16, 50, 129, 200], [1, 16, 3, 70, 33], heads, kv, D, 100)
        near(context(on(c, dev)), c, True)

    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("window", [1, 16, 60])
    def test_windows(self, dev, window):
        c = attention_case([64, 150, 20], [64, 70, 5], 8, 2, 64, 110, window)
        near(context(on(c, dev)), c, True)

    @pytest.mark.gpu
    @pytest.mark.parametrize("D", [64, 128])
    def test_split_keys(self, D):
        """Few queries behind long contexts: keys in parts, the sums merged."""
        c = attention_case([3000, 2500], [20, 9], 8, 2, D, 120)
        near(context(on(c, "cuda")), c, True)

    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("D", [64, 128])
    @pytest.mark.parametrize("window", [0, 1, 20])
    @pytest.mark.parametrize(
        "heads, kv, new",
        [(1, 1, [1, 16, 3, 0]), (1, 1, [32, 1, 5, 17]), (8, 2, [8, 2, 5, 1]), (8, 2, [4, 0, 1, 3]),
         (5, 1, [6, 6, 2, 1]), (16, 2, [4, 1, 3, 2]), (7, 1, [2, 4, 1, 3]), (22, 2, [2, 1, 2, 1]),
         (1, 1, [40, 16, 64, 33]), (8, 2, [10, 16, 9, 2]), (7, 1, [8, 9, 5, 1])],
    )
    def test_few_queries(self, dev, D, window, heads, kv, new):
        """As many as go beside one another in the columns of one product, of two, and of
        two blocks."""
        c = attention_case([40, 16, 177, 33], new, heads, kv, D, 150, window)
        near(context(on(c, dev)), c, True)

    @pytest.mark.gpu
    @pytest.mark.parametrize("D", [64, 128])
    @pytest.mark.parametrize("window", [0, 700])
    def test_few_queries_in_splits(self, D, window):
        """Long contexts beside short and empty ones, in parts that are merged."""
        c = attention_case([3000, 30, 2500, 5, 5], [5, 8, 3, 2, 0], 8, 2, D, 160, window)
        near(context(on(c, "cuda")), c, True)
        c["ctx"][3] = 0  # no keys: zeros
        d = on(c, "cuda")
        got = context(d)
        assert not got[16:18].any()
        near(got, c, True)

    @pytest.mark.gpu
    @pytest.mark.parametrize("window", [0, 1600])
    @pytest.mark.parametrize(
        "S, longest, most",
        [(64, 1535, 4), (64, 1536, 4), (65, 3100, 40), (257, 1800, 9), (300, 1600, 16)],
    )
    def test_few_queries_of_many_lengths(self, S, longest, most, window):
        """Long sequences among short ones and ones without queries."""
        g = torch.Generator().manual_seed(S)
        new = torch.randint(0, most + 1, (S,), generator=g)
        lens = new + torch.randint(0, 60, (S,), generator=g)
        at = torch.randperm(S, generator=g)[:5]
        lens[at] = torch.randint(longest // 2, longest + 1, (5,), generator=g)
        new[at[0]], lens[at[0]], lens[at[1]] = most, longest, longest
        c = attention_case(lens.tolist(), new.tolist(), 8, 8, 64, 165, window)
        near(context(on(c, "cuda")), c, True)

    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("n", [3, 70])
    def test_contexts_shorter_than_their_queries(self, dev, n):
        """Queries ahead of the context's first token see nothing: zeros."""
        c = attention_case([n, 90], [n, n], 8, 2, 64, 145)
        c["ctx"][0] = n - 2
        d = on(c, dev)
        got = context(d)
        assert not got[:2].any()
        near(got, c, True)

    @pytest.mark.gpu
    def test_sequences_without_queries(self):
        c = attention_case([64, 100, 40], [0, 7, 0], 8, 2, 128, 130)
        near(context(on(c, "cuda")), c, True)

    @pytest.mark.parametrize("dev", devices())
    def test_ids_outside_the_cache(self, dev):
        c = attention_case([40, 100], [9, 30], 8, 2, 128, 140)
        d = on(c, dev)
        d["table"][0] = torch.tensor([-5, 1 << 30, 3] + [0] * (d["table"].shape[1] - 3))
        d["ctx"][0] = 1 << 30
        got = context(d)
        near(got[9:], dict(c, q=c["q"][9:], cu=c["cu"][1:] - 9, ctx=c["ctx"][1:], table=c["table"][1:]), True)


def batch_oracle(lists, computed, new, rows, width, block):
    pos, slots, seqs, cu = [], [], [], [0]
    tables = []
    for s, (pages, c, n) in enumerate(zip(lists, computed, new)):
        for p in range(c, c + n):
            pos.append(p)
            slots.append(pages[p // block] * block + p % block if p // block < len(pages) else -1)
            seqs.append(s)
        cu.append(min(cu[-1] + n, rows))
        full = min(-(-(c + n) // block), len(pages))
        tables.append((pages[:full] + [0] * width)[:width])
    fill = max(0, rows - len(pos))
    return (
        (pos + [0] * fill)[:rows], (slots + [-1] * fill)[:rows], cu, tables,
        [c + n for c, n in zip(computed, new)], (seqs + [-1] * fill)[:rows],
    )


class TestBatch:
    def run(self, dev, lists, computed, new, rows, width, block):
        starts = [0]
        for x in lists:
            starts.append(starts[-1] + len(x))

        def vec(x):
            return torch.tensor(x, dtype=torch.int32, device=dev)

        got = ops.build_paged_batch(
            vec([i for x in lists for i in x]), vec(starts), vec(computed), vec(new), rows,
            width, block,
        )
        want = batch_oracle(lists, computed, new, rows, width, block)
        assert got.positions.dtype == torch.int64
        assert all(t.dtype == torch.int32 for t in got[1:])
        assert got.block_tables.shape == (len(lists), width)
        for g, w in zip(got, want):
            assert g.device.type == dev and g.tolist() == w

    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("block", [1, 4, 16, 100])
    @pytest.mark.parametrize(
        "computed, new, pad",
        [([0], [1], 0), ([0], [77], 3), ([5, 0, 160], [1, 0, 40], 0), ([0, 0], [0, 0], 0),
         ([0, 3, 0], [0, 9, 0], 5), ([], [], 4), ([], [], 0)],
    )
    def test_small(self, dev, computed, new, pad, block):
        g = torch.Generator().manual_seed(block)
        lists = [
            torch.randint(1, 1000, (-(-(c + n) // block) + i % 2,), generator=g).tolist()
            for i, (c, n) in enumerate(zip(computed, new))
        ]
        width = max([-(-(c + n) // block) for c, n in zip(computed, new)] + [0])
        self.run(dev, lists, computed, new, sum(new) + pad, width, block)

    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("S", [3, 1023, 1024, 1025, 2500])
    def test_many_requests(self, dev, S):
        """Past a block's chunk of lengths and of tokens."""
        g = torch.Generator().manual_seed(S)
        computed = torch.randint(0, 60, (S,), generator=g).tolist()
        new = torch.randint(0, 4 if S > 3 else 3000, (S,), generator=g).tolist()
        lists = [
            torch.randint(0, 1 << 20, (-(-(c + n) // PAGE),), generator=g).tolist()
            for c, n in zip(computed, new)
        ]
        width = max(len(x) for x in lists)
        self.run(dev, lists, computed, new, sum(new) + 11, width, PAGE)

    @pytest.mark.parametrize("dev", devices())
    def test_short_lists_and_rows(self, dev):
        """Tokens past their request's pages have no slot; rows and tables that are too
        short hold the first."""
        self.run(dev, [[7], [9, 8, 5]], [10, 0], [20, 40], 50, 2, PAGE)

    @pytest.mark.parametrize("dev", devices())
    def test_starts_out_of_range(self, dev):
        """Page lists that point outside stay inside."""

        def vec(x):
            return torch.tensor(x, dtype=torch.int32, device=dev)

        got = ops.build_paged_batch(vec([3, 4]), vec([-9, 1, 900]), vec([0, 0]), vec([20, 30]), 50, 3, PAGE)
        assert got.block_tables.tolist() == [[3, 0, 0], [4, 0, 0]]
        assert got.slot_mapping.tolist() == (
            list(range(48, 64)) + [-1] * 4 + list(range(64, 80)) + [-1] * 14
        )


class TestRefusals:
    """The same calls are refused on both sides."""

    @pytest.mark.parametrize("dev", devices())
    def test_batch(self, dev):
        def vec(x, dtype=torch.int32):
            return torch.tensor(x, dtype=dtype, device=dev)

        good = [vec([1, 2]), vec([0, 2]), vec([0]), vec([20]), 20, 2, PAGE]
        ops.build_paged_batch(*good)
        for i, bad in [
            (0, vec([1, 2], torch.int64)), (1, vec([0])), (1, vec([0, 1, 2])), (2, vec([0, 0])),
            (3, vec([[20]])), (3, vec([20], torch.int64)), (4, -1), (4, 1 << 31), (5, -1),
            (5, 1 << 31), (6, 0), (0, vec([1, 1, 2, 2])[::2]),
        ]:
            args = list(good)
            args[i] = bad
            with pytest.raises(RuntimeError):
                ops.build_paged_batch(*args)

    @pytest.mark.parametrize("dev", devices())
    def test_pages(self, dev):
        c = on(attention_case([20], [1], 4, 2, 64, 200), dev)
        k = torch.zeros((1, 2, 64), dtype=torch.bfloat16, device=dev)
        slots = torch.zeros(1, dtype=torch.int32, device=dev)
        scales = c["ks"].view(torch.uint8)
        for bad in [
            dict(ks=None), dict(vs=None), dict(ks=scales), dict(ks=scales[:1].view(E8M0)),
            dict(vs=scales.float()), dict(vc=c["vc"][:1]), dict(kc=c["kc"].float()),
        ]:
            x = dict(c, **bad)
            with pytest.raises(RuntimeError):
                decode(x)
            with pytest.raises(RuntimeError):
                context(x)
            with pytest.raises(RuntimeError):
                ops.reshape_and_cache(k, k, x["kc"], x["vc"], slots, k_scale=x["ks"], v_scale=x["vs"])
        for bad in [
            dict(q=c["q"][:, :3]), dict(q=c["q"][..., :32]), dict(table=c["table"].long()),
            dict(ctx=c["ctx"].long()), dict(window=-1),
            dict(kc=c["kc"][:0], vc=c["vc"][:0], ks=c["ks"][:0], vs=c["vs"][:0]),
        ]:
            with pytest.raises(RuntimeError):
                decode(dict(c, **bad))
            with pytest.raises(RuntimeError):
                context(dict(c, **bad), 1)
        for x, y, s in [(k, k[:, :1], slots), (k[..., :32], k[..., :32], slots), (k, k, slots[:0])]:
            with pytest.raises(RuntimeError):
                ops.reshape_and_cache(x, y, c["kc"], c["vc"], s, k_scale=c["ks"], v_scale=c["vs"])

    @pytest.mark.gpu
    def test_kernels_forms(self):
        """What the kernels do not take: other head sizes, larger groups, other types and
        devices."""
        c = on(attention_case([20], [1], 4, 2, 64, 210), "cuda")
        big = on(attention_case([20], [1], 18, 2, 64, 220), "cuda")
        with pytest.raises(RuntimeError):
            decode(big)  # nine heads to a KV head
        near(context(big), on(big, "cpu"), True)
        for bad in [
            dict(q=c["q"].half()), dict(q=c["q"].cpu()), dict(q=c["q"][:, :3]),
            dict(table=c["table"].long()), dict(table=c["table"][:0]), dict(ctx=c["ctx"].long()),
            dict(ctx=c["ctx"].cpu()), dict(window=-1), dict(kc=c["kc"][..., :32], vc=c["vc"][..., :32]),
        ]:
            with pytest.raises(RuntimeError):
                decode(dict(c, **bad))
            with pytest.raises(RuntimeError):
                context(dict(c, **bad), 1)
        with pytest.raises(RuntimeError):
            context(dict(c, cu=c["cu"].long()))
        k = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")
        slots = torch.zeros(2, dtype=torch.int32, device="cuda")
        for x, s in [(k, slots[:1]), (k, slots.long()), (k, slots.cpu()), (k.float(), slots), (k[:, :1], slots)]:
            with pytest.raises(RuntimeError):
                ops.reshape_and_cache(x, x, c["kc"], c["vc"], s, k_scale=c["ks"], v_scale=c["vs"])


def kinds(c, chunk):
    """A case's attention by decode, by few queries or by a chunk's kernel."""
    return context(c) if chunk else decode(c)


class TestScaleBytes:
    """Every byte a scale may have, at the ends of E8M0's range too.

    There bf16, in which pages are multiplied, has steps of 2^-133 below its normal
    numbers: a value may be off by half of one, 2^-134, which is
    - 2^-134 of the outputs (weights sum to 1), and once more where outputs are rounded;
    - of scores the sum of |q| 2^-134 times the scale, which moves a weight by that factor
      above and the denominator by it below."""

    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("least", [0, 1, 5])
    @pytest.mark.parametrize("new", [1, 4, 40])
    def test_least_scales(self, dev, new, least):
        g = torch.Generator().manual_seed(least)
        c = attention_case([50, 100], [min(new, 40), new], 8, 2, 128, 230)
        for n in ("ks", "vs"):
            e = least + torch.randint(0, 3, c[n].shape, generator=g)
            c[n] = e.to(torch.uint8).view(E8M0)
        # scores of a few units all the same
        c["scale"] = 2.0 ** (110 - least)
        got = kinds(on(c, dev), new > 1)
        out, off, size = attention_oracle(c)
        lost = 2.0**-134
        moved = 2 * c["q"].double().abs().sum(-1, keepdim=True) * c["scale"] * lost
        off = off + 2 * lost + moved * size + (2.0**-8 * size if new > 1 else 0)
        # (the bound tells 2^-127 from 2^-126)
        assert float((off / out.abs().amax(-1, keepdim=True)).max()) < 0.1
        assert bool(((got.double().cpu() - out).abs() <= off).all())

    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("new", [1, 4, 40])
    @pytest.mark.parametrize("which", ["ks", "vs"])
    def test_no_number(self, dev, new, which):
        """Byte 255: what sees the page is no number, nothing else is touched."""
        c = attention_case([50, 100], [new, new], 8, 2, 64, 240)
        page = int(c["table"][0, 0])
        c["vc"].view(torch.uint8)[page, 1] = 56  # (one sign: as infinities they would add up)
        c[which].view(torch.uint8)[page, 1] = 255
        got = kinds(on(c, dev), new > 1).cpu()
        # query heads 4 to 7 read KV head 1
        assert bool(got[:new, 4:].isnan().all())
        assert not got[:new, :4].isnan().any() and not got[new:].isnan().any()
        c[which].view(torch.uint8)[page, 1] = 120
        out, off, size = attention_oracle(c)
        off = off + (2.0**-8 * size if new > 1 else 0)
        near_by = (got.double() - out).abs() <= off
        assert bool(near_by[:new, :4].all()) and bool(near_by[new:].all())


class TestAheadOfTheWindow:
    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("D", [64, 128])
    @pytest.mark.parametrize(
        "window, new",
        [(1, 1), (20, 1), (48, 1), (3, 5), (40, 5), (1, 40), (20, 40), (65, 40), (100, 150), (90, 77)],
    )
    def test_may_be_anything(self, dev, D, window, new):
        """Keys that no query of their sequence sees, in whole pages and in part of one: bytes
        and scales that are no numbers, pages that are not the sequence's."""
        lens = [max(new, 30), 300, 173]
        c = attention_case(lens, [new] * 3, 8, 2, D, 250, window)
        near(kinds(on(c, dev), new > 1), c, new > 1)
        for i, n in enumerate(lens):
            low = max(n - new - window + 1, 0)
            pages, rows = c["table"][i, : low // PAGE].long(), low % PAGE
            for scale, cache in (("ks", "kc"), ("vs", "vc")):
                c[scale].view(torch.uint8)[pages] = 255
                c[cache].view(torch.uint8)[c["table"][i, low // PAGE], :, :rows] = 0x7F
            c["table"][i, : low // PAGE // 2] = -7
        # (page 0, where those now point, is nobody's)
        c["ks"].view(torch.uint8)[0] = c["vs"].view(torch.uint8)[0] = 255
        d = dict(c, table=c["table"].clamp(min=0))
        for n in ("kc", "vc"):  # the oracle's: numbers, which it gives no weight
            raw = c[n].view(torch.uint8).clone()
            raw[raw % 128 == 127] = 0
            d[n] = raw.view(E4M3)
        for n in ("ks", "vs"):
            raw = c[n].view(torch.uint8).clone()
            raw[raw == 255] = 118
            d[n] = raw.view(E8M0)
        near(kinds(on(c, dev), new > 1), d, new > 1)


class TestWindowsInWideTables:
    @pytest.mark.gpu
    @pytest.mark.parametrize("S", [1, 5, 13, 25, 70])
    @pytest.mark.parametrize("window", [1, 255, 500, 1000, 2500])
    def test_few_sequences(self, S, window):
        """In one part and in several, by what the window reaches."""
        g = torch.Generator().manual_seed(S)
        lens = torch.randint(1, 3000, (S,), generator=g)
        lens[0], lens[-1] = window + 17, 2999
        c = attention_case(lens.tolist(), [1] * S, 8, 8, 64, 270, window)
        c["table"] = torch.nn.functional.pad(c["table"], (0, 900))
        near(decode(on(c, "cuda")), c)


class TestWindowsPastTheTables:
    @pytest.mark.parametrize("dev", devices())
    @pytest.mark.parametrize("new", [1, 5, 70])
    @pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 60, 1000])
    def test_hide_nothing(self, dev, new, window):
        """The results are those without a window; of contexts shorter than their queries too,
        whose first ones stand ahead of position 0."""
        c = attention_case([70, 300, 90], [new] * 3, 8, 2, 64, 260)
        c["ctx"][2] = max(new - 4, 1)
        d = on(c, dev)
        got = kinds(dict(d, window=window), new > 1)
        near(got, c, new > 1)
        assert torch.equal(got, kinds(d, new > 1))


class TestLongParts:
    """Parts of more keys than a wave holds page ids and scales for (4096: 64 tiles of the
    chunk kernel, 32 pairs of pages of each of four waves), which it fetches anew."""

    def parts(self, c):
        """Key parts that such a call is cut into."""
        import ctypes

        rule = ctypes.CDLL(ops._C.__file__).ks_context_scaled_splits
        rule.argtypes = [ctypes.c_int, ctypes.c_long] + [ctypes.c_int] * 5
        S, longest = len(c["ctx"]), int((c["cu"][1:] - c["cu"][:-1]).max())
        H, kv = c["q"].shape[1], c["kc"].shape[1]
        return rule(S, c["q"].shape[0] * H, longest, H, kv, c["table"].shape[1], c["window"])

    def check(self, c, heads):
        """By some KV heads (and one query head of each)."""
        got = context(on(c, "cuda"))
        G = c["q"].shape[1] // c["kc"].shape[1]
        some = torch.tensor(heads)
        few = dict(c, q=c["q"][:, some * G])
        for n in ("kc", "vc", "ks", "vs"):
            few[n] = c[n].view(torch.uint8)[:, some].contiguous().view(c[n].dtype)
        near(got[:, some * G], few, True)

    @pytest.mark.gpu
    @pytest.mark.parametrize("D, kv, window", [(64, 128, 0), (64, 128, 5003), (128, 128, 8200)])
    def test_chunks_in_one_part(self, D, kv, window):
        c = attention_case([9001], [512], kv, kv, D, 280, window)
        assert self.parts(c) == 1
        self.check(c, [0, 77, 127])

    @pytest.mark.gpu
    @pytest.mark.parametrize("window", [0, 139000])
    def test_chunks_in_several(self, window):
        c = attention_case([140003], [70], 2, 1, 64, 290, window)
        c["table"] = c["table"][:, :8751].contiguous()
        assert self.parts(c) * 4096 < min(140003, window or 140003)
        self.check(c, [0])

    @pytest.mark.gpu
    @pytest.mark.parametrize("D", [64, 128])
    @pytest.mark.parametrize("window", [0, 6005])
    @pytest.mark.parametrize("most", [4, 20, 40])
    def test_few_queries_in_one_part(self, D, window, most):
        g = torch.Generator().manual_seed(most)
        new = torch.randint(1, most + 1, (32,), generator=g)
        lens = new + torch.randint(0, 60, (32,), generator=g)
        lens[3], lens[20], lens[31], new[20] = 9001, 4130, 12345, most
        c = attention_case(lens.tolist(), new.tolist(), 8, 8, D, 300, window)
        assert self.parts(c) == 1
        self.check(c, [0, 5])

    @pytest.mark.gpu
    @pytest.mark.parametrize("window", [0, 18001])
    def test_few_queries_in_several(self, window):
        lens = [40 + i for i in range(16)]
        lens[2] = 20007
        c = attention_case(lens, [3] * 16, 16, 8, 64, 310, window)
        assert self.parts(c) == 2
        self.check(c, [0, 7])


class TestLongWrites:
    @pytest.mark.gpu
    @pytest.mark.parametrize(
        "T, kv, D, order",
        [(2048, 9, 64, "runs"), (2049, 9, 64, "runs"), (5000, 8, 128, "any"), (8191, 4, 128, "runs"),
         (9001, 9, 64, "twice"), (70001, 5, 64, "runs"), (66000, 1, 64, "any")],
    )
    def test_is_the_plain_form(self, T, kv, D, order):
        """Prompts of more tokens than a block has, in several blocks to a page, whose slots
        stand in runs, in any order, and twice; of a slot map at an odd address too."""
        g = torch.Generator().manual_seed(T)
        pages = T // PAGE + 40
        kc, ks = make_cache(pages, kv, D, 16)
        x = (torch.randn((T, 2 * kv, D), generator=g) * torch.exp(torch.randn((T, 1, 1), generator=g)))
        x = x.to(torch.bfloat16)
        if order == "runs":  # one sequence, from inside a page on
            ids = torch.randperm(pages, generator=g)
            at = torch.arange(T) + 5
            slots = ids[at // PAGE] * PAGE + at % PAGE
        elif order == "any":
            slots = torch.randperm(pages * PAGE, generator=g)[:T]
        else:
            slots = torch.randint(-5, pages * PAGE + 5, (T,), generator=g)
        slots = slots.int()
        outs = []
        for dev, skip in (("cpu", 0), ("cuda", 0), ("cuda", 1)):
            c = [t.view(torch.uint8).to(dev).clone().view(t.dtype) for t in (kc, kc, ks, ks)]
            sl = torch.cat([slots[:skip], slots]).to(dev)[skip:]
            y = x.to(dev)
            ops.reshape_and_cache(y[:, :kv], y[:, kv:], c[0], c[1], sl, k_scale=c[2], v_scale=c[3])
            outs.append([t.view(torch.uint8).cpu() for t in c])
        for got in outs[1:]:
            for a, b in zip(got, outs[0]):
                assert torch.equal(a, b)
