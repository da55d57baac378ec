"""``process_logits`` and ``next_tokens`` against the written formulas, in 64
bits for the sums and word by word for the random numbers."""

from __future__ import annotations

import importlib
import math

import numpy as np
import pytest
import torch

from src.kernels.logits import next_tokens, process_logits

pytestmark = pytest.mark.gpu

INF = float("inf")


def case(B, V, T, dtype, seed=0, bias=None, mask=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    a = {"logits": (torch.randn(B, V, generator=g, device="cuda") * 3).to(dtype)}
    if T is not None:
        a["tokens"] = (rand(B, T) ** 3 * V).long().clamp(max=V - 1)
        a["lengths"] = (rand(B) * (T + 1)).long().clamp(max=T)
        a["prompt_lengths"] = (rand(B) * (T + 1) * 0.5).long()
        a["repetition_penalty"] = 1 + rand(B)
        a["presence_penalty"] = rand(B)
        a["frequency_penalty"] = rand(B) * 0.5
    if bias is not None:
        a["bias"] = torch.randn(*((V,) if bias == "shared" else (B, V)), generator=g, device="cuda")
    if mask is not None:
        words = -(-V // 32)
        a["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (words,) if mask == "shared" else (B, words), generator=g,
                                     device="cuda", dtype=torch.int64).to(torch.int32)
    return a


def adjusted(a, real=np.float32):
    """The formula, row by row in numpy; in fp32 every operation is rounded
    once, as documented."""
    z = a["logits"].float().cpu().numpy().astype(real)
    B, V = z.shape
    row = lambda name, b, neutral: real(neutral if a.get(name) is None else a[name] if not isinstance(  # noqa: E731
        a[name], torch.Tensor) else a[name][b].item())
    for b in range(B):
        if a.get("tokens") is not None:
            T = a["tokens"].shape[1]
            n = T if a.get("lengths") is None else min(max(int(a["lengths"][b]), 0), T)
            p = 0 if a.get("prompt_lengths") is None else min(max(int(a["prompt_lengths"][b]), 0), n)
            h = a["tokens"][b].cpu().numpy()
            r = row("repetition_penalty", b, 1)
            fit = lambda t: t[(t >= 0) & (t < V)]  # noqa: E731
            seen = np.unique(fit(h[:n]))
            z[b, seen] = np.where(z[b, seen] > 0, z[b, seen] / r, z[b, seen] * r)
            gen, count = np.unique(fit(h[p:n]), return_counts=True)
            z[b, gen] = z[b, gen] - row("frequency_penalty", b, 0) * count.astype(real)
            z[b, gen] = z[b, gen] - row("presence_penalty", b, 0)
        if a.get("bias") is not None:
            z[b] = z[b] + (a["bias"] if a["bias"].dim() == 1 else a["bias"][b]).float().cpu().numpy().astype(real)
        if a.get("allowed") is not None:
            w = (a["allowed"] if a["allowed"].dim() == 1 else a["allowed"][b]).contiguous().cpu().numpy()
            z[b, np.unpackbits(w.view(np.uint8), bitorder="little")[:V] == 0] = -np.inf
    return z


def noise(seed, position, V):
    """-log(-log u), the generator's words as Python integers."""
    out = []
    for i in range(0, V, 4):
        c, k = [i // 4, position & 0xFFFFFFFF, (position >> 32) & 0xFFFFFFFF, 0], [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
        for _ in range(7):
            x, y = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(y >> 32) ^ c[1] ^ k[0], y & 0xFFFFFFFF, (x >> 32) ^ c[3] ^ k[1], x & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        out += [-math.log(-math.log1p(-(w + 0.5) * 2.0 ** -32)) for w in c]
    return np.array(out[:V])


def check_process(a, **kw):
    got = process_logits(**a, **kw)
    want = torch.from_numpy(adjusted(a)).to(got.dtype)
    assert got.dtype == (kw["out"].dtype if "out" in kw else a["logits"].dtype)
    assert torch.equal(got.cpu().float().nan_to_num(nan=12345.0), want.float().nan_to_num(nan=12345.0))
    return got


def check_next(a, temperature=None, seeds=None, positions=None):
    ids, lp = next_tokens(**a, temperature=temperature, seeds=seeds, positions=positions)
    z = adjusted(a)
    B, V = z.shape
    assert ids.shape == lp.shape == (B,) and ids.dtype == torch.int64 and lp.dtype == torch.float32
    for b in range(B):
        t = 0.0 if temperature is None else float(temperature if not isinstance(temperature, torch.Tensor)
                                                  else temperature[b])
        zt = z[b].astype(np.float64) / (t if t > 0 else 1.0)
        score = zt
        if t > 0 and np.isfinite(zt.max()):  # relative to the largest: 1e38 has no bits for the noise
            score = zt - zt.max() + noise(int(seeds[b]), 0 if positions is None else int(positions[b]), V)
        want = int(np.argmax(score))  # the first of equals; a NaN above all
        assert int(ids[b]) == want, (b, int(ids[b]), want)
        top = zt.max()
        if np.isneginf(top):
            assert float(lp[b]) == -INF and want == 0
            continue
        if not np.isfinite(top):
            assert math.isnan(float(lp[b]))
            continue
        exact = zt[want] - top - math.log(np.exp(zt - top).sum())
        # (z - top) / t and the logarithm, half a place each of their
        # magnitudes; the exponentials' arguments are off by up to 3 half
        # places of |z - top| / t <= 104 (beyond, they vanish), the
        # approximated exponential by 2 places, each thread's and CTA's sum by
        # half a place an addition: at most 32 + 40 deep per 65,536 logits
        far = min(float(np.abs(zt[np.isfinite(zt)] - top).max()), 104.0)
        terms = 32 * -(-V // 65536) + 40
        tol = (abs(zt[want] - top) * 2 + abs(exact) + far * 2 + 4 + terms) * 2.0 ** -24 * 2
        assert abs(float(lp[b]) - exact) <= tol, (b, float(lp[b]), exact)
    return ids, lp


@pytest.mark.parametrize("V", [1, 7, 31, 32, 33, 255, 257, 1000, 6305, 50277])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_process(V, dtype):
    for B, T, bias, mask in ((1, 40, None, None), (3, 0, "row", "shared"), (5, 300, "shared", "row"),
                             (2, None, None, "row"), (2, None, None, None)):
        a = case(B, V, T, dtype, seed=V + B, bias=bias, mask=mask)
        check_process(a)
        check_process(a, out=torch.empty(B, V, device="cuda", dtype=torch.float32))


@pytest.mark.parametrize("V", [1, 7, 33, 255, 257, 1000, 6305])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_next(V, dtype):
    for B, T, bias, mask in ((1, 40, None, None), (3, 0, "row", "shared"), (4, 300, "shared", "row"),
                             (2, None, None, None)):
        a = case(B, V, T, dtype, seed=V + B, bias=bias, mask=mask)
        check_next(a)
        g = torch.Generator(device="cuda").manual_seed(V)
        seeds = torch.randint(-2 ** 63, 2 ** 63 - 1, (B,), generator=g, device="cuda")
        pos = torch.randint(0, 2 ** 40, (B,), generator=g, device="cuda")
        temp = torch.rand(B, generator=g, device="cuda") + 0.25
        temp[0] = 0.0  # one greedy row among them
        check_next(a, temp, seeds, pos)
        check_next(a, 1.0, seeds)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_vocabulary_of_several_rounds(dtype):
    a = case(2, 140001, 900, dtype, seed=4, mask="row")
    a["tokens"][0, :5] = torch.tensor([0, 65535, 65536, 131072, 140000])
    a["lengths"][:] = 900
    check_process(a)
    check_next(a)
    check_next(a, 0.7, torch.tensor([3, -9], device="cuda"))


@pytest.mark.parametrize("temperature", [1e-30, 1e-3, 0.05, 3.0, 100.0, 1e30])
def test_temperatures(temperature):
    a = case(4, 3001, None, torch.float32, seed=8)
    seeds = torch.arange(4, device="cuda") * 7919 + 2 ** 33
    check_next(a, temperature, seeds)


def test_one_dominant_token():
    """The winner's own noise can be large: the screen must still keep it."""
    a = {"logits": torch.full((256, 777), -40.0, device="cuda")}
    a["logits"][:, 500] = 5.0
    seeds = torch.arange(256, device="cuda") + 10 ** 12
    ids, lp = check_next(a, 1.0, seeds)
    assert bool((ids == 500).all())


def test_draws_follow_the_distribution():
    """4096 draws from four tokens: counts within five standard deviations."""
    p = torch.tensor([0.5, 0.25, 0.15, 0.1])
    n = 4096
    logits = p.log().cuda().expand(n, 4)
    ids, _ = next_tokens(logits, temperature=1.0, seeds=torch.full((n,), 42, device="cuda"),
                         positions=torch.arange(n, device="cuda"))
    count = torch.bincount(ids.cpu(), minlength=4).double()
    assert bool(((count - n * p).abs() <= 5 * (n * p * (1 - p)).sqrt()).all()), count


def test_ties_go_to_the_lowest_index():
    z = torch.zeros(4, 50280, device="cuda", dtype=torch.bfloat16)
    z[1, 49999], z[1, 6303], z[1, 6304] = 2.0, 2.0, 2.0
    z[2, :] = -0.0
    z[2, 30000] = 0.0  # -0 and 0 are equal
    z[3, 50279] = 1.0
    ids, _ = next_tokens(z)
    assert ids.tolist() == [0, 6303, 0, 50279]


@pytest.mark.parametrize("sample", [False, True])
def test_values_that_are_not_finite(sample):
    V = 20000
    z = torch.randn(8, V, device="cuda")
    z[0] = -INF                                          # nothing left
    z[1, 17000], z[1, 900] = float("nan"), INF           # NaN above infinity
    z[2, 300], z[2, 19999] = INF, INF                    # first infinity
    z[3, 5:] = -INF
    z[4, 19000], z[4, 20] = float("nan"), float("nan")
    z[5, :] = torch.finfo(torch.float32).min             # masked by the lowest value
    z[5, 777] = -3e38
    z[6, :] = torch.finfo(torch.float32).min
    allowed = torch.full((8, 625), -1, dtype=torch.int32, device="cuda")
    allowed[7] = 0                                       # the mask leaves nothing
    z[7, 4] = float("nan")                               # NaN in a masked place
    a = {"logits": z, "allowed": allowed}
    kw = dict(temperature=1.0, seeds=torch.arange(8, device="cuda")) if sample else {}
    ids, lp = next_tokens(**a, **kw)
    assert int(ids[0]) == 0 and float(lp[0]) == -INF
    assert int(ids[1]) == 17000 and math.isnan(float(lp[1]))
    assert int(ids[2]) == 300 and math.isnan(float(lp[2]))
    assert int(ids[4]) == 20 and math.isnan(float(lp[4]))
    assert int(ids[7]) == 0 and float(lp[7]) == -INF
    keep = [3, 5, 6]
    rows = {"logits": z[keep], "allowed": allowed[keep]}
    if sample:
        check_next(rows, 1.0, torch.tensor(keep, device="cuda"))
        assert ids[keep].tolist() == next_tokens(**rows, temperature=1.0,
                                                 seeds=torch.tensor(keep, device="cuda"))[0].tolist()
    else:
        check_next(rows)
    check_process(a)


def test_histories():
    """Lengths of 0, past the end and negative, prompts longer than the
    history, ids that are padding, one token many times, int32 everywhere."""
    V, T = 500, 5000
    a = case(6, V, T, torch.float32, seed=2)
    a["lengths"][:] = torch.tensor([0, T + 5, -3, 100, T, 1], device="cuda")
    a["prompt_lengths"][:] = torch.tensor([0, 10, 5, 4000, -7, 1], device="cuda")
    a["tokens"][1, ::7] = -1
    a["tokens"][1, 1::7] = V
    a["tokens"][1, 2::7] = 2 ** 40
    a["tokens"][4] = 123
    check_process(a)
    check_next(a)
    b = dict(a, tokens=a["tokens"].clamp(-5, V + 5).int(), lengths=a["lengths"].int(),
             prompt_lengths=a["prompt_lengths"].int())
    check_process(b)
    c = {k: v for k, v in b.items() if k not in ("lengths", "prompt_lengths")}
    check_process(c)
    check_next(dict(c, repetition_penalty=1.3, presence_penalty=0.2, frequency_penalty=-0.1))
    check_process(dict(c, repetition_penalty=None, presence_penalty=None, frequency_penalty=None))
    check_process(dict(c, repetition_penalty=2.0, presence_penalty=None, frequency_penalty=None))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(dtype):
    wide = torch.randn(6, 2101, device="cuda").to(dtype)
    hist = torch.randint(0, 999, (6, 90), device="cuda")
    kw = dict(repetition_penalty=1.5, frequency_penalty=0.25)
    for x, t in ((wide[:, :1000], hist), (wide[:, 1:1001], hist[:, 3:50]), (wide[::2, 3:2000], hist[::2]),
                 (torch.randn(1000, 6, device="cuda").to(dtype).t(), hist),
                 (wide[:1, :1000].expand(6, 1000), hist[:1].expand(6, 90)),
                 (wide[:, 8:1008], torch.randint(0, 999, (90, 6), device="cuda").t())):
        a = dict(logits=x, tokens=t, **kw)
        check_process(a)
        check_next(a)
        out = torch.full((x.shape[0], x.shape[1] + 9), 7.0, device="cuda", dtype=dtype)
        check_process(a, out=out[:, 4:-5])
        assert bool((out[:, :4] == 7).all()) and bool((out[:, -5:] == 7).all())
    a = dict(logits=wide[:, :999], bias=torch.randn(6, 2000, device="cuda")[:, 1:1000].bfloat16(),
             allowed=torch.randint(-2 ** 31, 2 ** 31, (40, 6), device="cuda").int().t())
    check_process(a)
    check_next(a)
    check_process(dict(a, bias=torch.randn(999, device="cuda", dtype=torch.float64)))


def test_in_place():
    a = case(3, 1000, 50, torch.bfloat16, seed=1, mask="row")
    want = torch.from_numpy(adjusted(a)).bfloat16()
    got = process_logits(**a, out=a["logits"])
    assert got is a["logits"] and torch.equal(got.cpu(), want)


def test_offsets_past_32_bits():
    B, V = 44000, 50280  # 2.2e9 logits
    z = torch.zeros(B, V, device="cuda", dtype=torch.bfloat16)
    z[-1, 50000], z[-1, 17], z[0, 3] = 3.0, 5.0, 1.0
    hist = torch.full((B, 1), 17, device="cuda", dtype=torch.int32)
    ids, _ = next_tokens(z, hist, presence_penalty=4.0)
    assert int(ids[-1]) == 50000 and int(ids[0]) == 3
    process_logits(z, hist, presence_penalty=4.0, out=z)
    assert float(z[-1, 17]) == 1.0 and float(z[-1, 50000]) == 3.0 and float(z[1, 17]) == -4.0


def test_nothing_to_do():
    z = torch.empty(0, 100, device="cuda")
    assert process_logits(z).shape == (0, 100)
    ids, lp = next_tokens(z)
    assert ids.shape == lp.shape == (0,)
    assert process_logits(torch.empty(3, 0, device="cuda")).shape == (3, 0)


def test_same_bits_on_every_run_and_stream():
    a = case(9, 50280, 400, torch.bfloat16, seed=6, bias="row", mask="row")
    kw = dict(temperature=0.8, seeds=torch.arange(9, device="cuda"))
    ids, lp = next_tokens(**a, **kw)
    z = process_logits(**a)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([(*next_tokens(**a, **kw), process_logits(**a)) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(x[0], ids) and torch.equal(x[1], lp) and torch.equal(x[2], z) for run in got for x in run)


def test_captured():
    """A captured draw goes on by its position tensor."""
    a = case(4, 5000, 64, torch.float32, seed=9)
    seeds, pos = torch.arange(4, device="cuda"), torch.zeros(4, dtype=torch.long, device="cuda")
    next_tokens(**a, temperature=1.0, seeds=seeds, positions=pos)
    process_logits(**a)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ids, lp = next_tokens(**a, temperature=1.0, seeds=seeds, positions=pos)
        z = process_logits(**a)
        pos += 1
    drawn = []
    for t in range(3):
        a["logits"].normal_()
        want = next_tokens(**a, temperature=1.0, seeds=seeds, positions=torch.full((4,), t, device="cuda"))
        g.replay()
        assert torch.equal(ids, want[0]) and torch.equal(lp, want[1]) and torch.equal(z, process_logits(**a))
        drawn.append(ids.tolist())
    assert int(pos[0]) == 3


def test_refusals():
    z = torch.zeros(2, 100, device="cuda")
    hist = torch.zeros(2, 5, dtype=torch.long, device="cuda")
    bad = [dict(logits=z.half()), dict(logits=z[0]), dict(tokens=hist[:1]), dict(tokens=hist.float()),
           dict(tokens=hist.cpu()), dict(lengths=hist[:, 0]), dict(tokens=hist, lengths=hist[0]),
           dict(tokens=hist, repetition_penalty=torch.ones(3, device="cuda")), dict(bias=torch.zeros(99, device="cuda")),
           dict(bias=torch.zeros(3, 100, device="cuda")), dict(allowed=torch.zeros(3, dtype=torch.int32, device="cuda")),
           dict(allowed=torch.zeros(4, device="cuda")), dict(tokens=hist, presence_penalty=torch.ones(2))]
    for kw in bad:
        for f in (process_logits, next_tokens):
            with pytest.raises(AssertionError):
                f(**dict(dict(logits=z), **kw))
    for f in (process_logits, next_tokens):
        with pytest.raises(ValueError):
            f(z, hist, repetition_penalty=0.0)
        with pytest.raises(RuntimeError):
            f(z.clone().requires_grad_())
    for kw in (dict(temperature=1.0), dict(temperature=1.0, seeds=torch.zeros(2, dtype=torch.int32, device="cuda")),
               dict(temperature=1.0, seeds=hist[:, 0], positions=hist[0])):
        with pytest.raises(AssertionError):
            next_tokens(z, **kw)
    with pytest.raises(AssertionError):
        next_tokens(torch.empty(2, 0, device="cuda"))
    for out in (z[:, :50], torch.empty(2, 100, device="cuda").half(), torch.empty(1, 100, device="cuda").expand(2, 100),
                z.flatten()[1:].as_strided((2, 99), (99, 1)), torch.empty(2, 100)):
        with pytest.raises(AssertionError):
            process_logits(z[:, :out.shape[1]] if out.shape[1] == 99 else z, out=out)


@pytest.mark.parametrize("V", [600, 60000])
@pytest.mark.parametrize("T", [3000, 16384, 16385, 70000])
def test_long_histories(V, T):
    """Past what a thread holds, past 16-bit counters, in several windows."""
    a = case(2, V, T, torch.float32, seed=T, mask="row")
    a["lengths"][:] = T
    a["prompt_lengths"][:] = torch.tensor([0, T // 2], device="cuda")
    a["tokens"][0, : T - 100] = V - 1
    check_process(a)
    check_process(dict(a, logits=a["logits"].bfloat16()))
    check_next(a)
    check_next(a, 0.9, torch.tensor([5, 6], device="cuda"))


@pytest.mark.parametrize("python_path", [False, True])
def test_host_module_and_python_path_agree(python_path, monkeypatch):
    """The host module serves the ordinary calls; both ways are the formula."""
    from src import _native as nat
    mod = importlib.import_module("src.kernels.logits")
    assert nat.host_entry("next_tokens") is not nat._no_host, "lib/m3_host.so is not built"
    if python_path:
        monkeypatch.setattr(mod, "_host_process", nat._no_host)
        monkeypatch.setattr(mod, "_host_next", nat._no_host)
    seeds, pos = torch.arange(4, device="cuda"), torch.arange(4, device="cuda") + 2 ** 35
    for bias, mask in ((None, None), ("row", "shared"), ("shared", "row")):
        a = case(4, 1000, 60, torch.float32, seed=11, bias=bias, mask=mask)
        a["logits"] = a["logits"][:, :991]
        a["tokens"] = a["tokens"].clamp(max=990)
        if bias:
            a["bias"] = a["bias"][..., :991]
        check_process(a)
        check_next(a)
        check_next(a, 0.8, seeds, pos)
        check_next(dict(a, repetition_penalty=1.25, presence_penalty=0.5, frequency_penalty=None), 0.8, seeds)
        b = dict(a, lengths=a["lengths"].int(), prompt_lengths=None, tokens=a["tokens"].int())
        check_process(b)


def test_host_module_leaves_what_it_does_not_take():
    from src import _native as nat
    f = nat.host_entry("process_logits")
    z, hist = torch.zeros(2, 100, device="cuda"), torch.zeros(2, 5, dtype=torch.long, device="cuda")
    none = [None] * 8
    assert f(z, *none) is not None
    for args in ((z.half(), *none), (z[0], *none), (z.t().contiguous().t(), *none), (z[:0], *none), (z.cpu(), *none),
                 (z.clone().requires_grad_(), *none), (z, hist[:1], *none[1:]), (z, hist.float(), *none[1:]),
                 (z, None, hist[:, 0].contiguous(), *none[2:]), (z, hist, None, None, 0.0, *none[4:]),
                 (z, hist, None, None, torch.ones(3, device="cuda"), *none[4:]), (z, *none[:6], torch.zeros(99, device="cuda"), None),
                 (z, *none[:7], torch.zeros(3, dtype=torch.int32, device="cuda")), (z, *none[:7])):
        assert f(*args) is None
    g = nat.host_entry("next_tokens")
    assert g(z, *none, 1.0, None, None) is None and g(z, *none, 1.0, torch.zeros(2, dtype=torch.int32, device="cuda"), None) is None


def test_infinite_temperature_is_uniform():
    z = torch.full((2000, 8), -INF, device="cuda")
    z[:, :4] = torch.tensor([0.0, 5.0, -3.0, 100.0], device="cuda")
    ids, lp = next_tokens(z, temperature=float("inf"), seeds=torch.arange(2000, device="cuda"))
    count = torch.bincount(ids.cpu(), minlength=8)
    assert not count[4:].any() and bool(((count[:4] - 500.0).abs() <= 5 * (2000 * 0.25 * 0.75) ** 0.5).all())
    torch.testing.assert_close(lp, torch.full_like(lp, -math.log(4.0)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [20000, 20003])
def test_in_place_of_many_rows(V, dtype):
    """Seen logits are read before any thread stores over them."""
    for T in (30, 1500, 6000):
        a = case(300, V, T, dtype, seed=T, mask="shared")
        want = process_logits(**a)
        for _ in range(3):
            b = dict(a, logits=a["logits"].clone())
            assert torch.equal(process_logits(**b, out=b["logits"]), want)
        small = {k: v[:3] if v.shape[0] == 300 else v for k, v in a.items()}
        check_process(small)
        check_next(small)
