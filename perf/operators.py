"""Timed cases of the language-model operators: products with 4-bit weights,
and what a decode step does with its logits.

Three operators, each with the smallest, ordinary and largest calls that a
token step of ``Mamba3LMDecoder`` makes of it:

``linear_w4``       y = x W^T with W[n, k] = (code - zero) * scale, one scale
                    (and zero) per row and group of 32, 64 or 128 columns;
                    x (M, K) holds the batch rows of a decode step.
``process_logits``  penalties for repeated tokens, a bias and a bit mask of
                    allowed tokens, applied to (B, V) logits.
``next_tokens``     the same adjustments, then the next token of every row
                    (largest logit, or drawn by its row's seed and position)
                    with its log-probability, the adjusted logits not stored.

With ``own`` false, ``run`` computes them with elementary torch operations in
32 bits (64 for the random scores); with ``own`` true it calls the
``src.kernels`` entry points.

4-bit storage: blocks of 16 rows by 128 columns (both padded) follow each
other along a row of blocks: codes (ceil(N / 16), ceil(K / 128), 16, 16) int32.
Word 4 t + j of a block's row holds its columns 32 j + 8 t .. + 7: column + 0,
2, 4, 6 in bits 0, 4, 8, 12 and column + 1, 3, 5, 7 in bits 16, 20, 24, 28.
"""

import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NIBBLE_SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)  # of columns + 0 .. + 7
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# counter-based generator (Salmon et al., "Parallel random numbers: as easy as
# 1, 2, 3", SC 2011): multipliers and key increments of its 4 x 32 bit form
PHILOX_M = (0xD2511F53, 0xCD9E8D57)
PHILOX_W = (0x9E3779B9, 0xBB67AE85)
PHILOX_ROUNDS = 7


def kernels():
    """The framework's entry points."""
    pkg = os.path.join(ROOT, "mamba3-fused-triton-kernel_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import src.kernels as k
    return k


def listed():
    w4 = {"op": "linear_w4"}
    pl = {"op": "process_logits"}
    nt = {"op": "next_tokens"}
    return [
        # in_proj of the d_model 256 MIMO rank-4 layer, one sequence: latency
        dict(w4, name="w4_d256_b1_f32", M=1, N=1600, K=256, G=32, x="f32", s="f32", zeros=False),
        # in_proj of the d_model 2048 stack's layer, one bf16 sequence: the weight stream
        dict(w4, name="w4_d2048_inproj_b1", M=1, N=9440, K=2048, G=128, x="bf16", s="bf16", zeros=False),
        # its out_proj for a small batch, finer groups with zero points
        dict(w4, name="w4_d2048_outproj_b16", M=16, N=2048, K=4096, G=64, x="bf16", s="bf16", zeros=True),
        # an odd layer in fp32 (ragged rows, columns and last group)
        dict(w4, name="w4_odd_b5_f32", M=5, N=4099, K=1111, G=128, x="f32", s="f32", zeros=True),
        # the LM head of the default language model for the largest small batch
        dict(w4, name="w4_lmhead_b64", M=64, N=50280, K=2560, G=128, x="bf16", s="bf16", zeros=False),
        # one sequence with a short history: every penalty, fp32 logits
        dict(pl, name="logits_b1_f32", B=1, V=50280, T=200, dtype="f32", penalties=True, bias="none", mask="none"),
        # grammar-constrained rows over a vocabulary that is no multiple of anything
        dict(pl, name="logits_b37_odd_f32", B=37, V=50277, T=777, dtype="f32", penalties=True, bias="row",
             mask="row"),
        # a large serving batch with long histories, one bias and one mask for all
        dict(pl, name="logits_b256_bf16", B=256, V=50280, T=2048, dtype="bf16", penalties=True, bias="shared",
             mask="shared"),
        # greedy decoding of one sequence
        dict(nt, name="next_b1_greedy_f32", B=1, V=50280, T=0, dtype="f32", penalties=False, bias="none",
             mask="none", sample=False),
        # sampling for an ordinary batch with penalties and a mask per row
        dict(nt, name="next_b32_sample_f32", B=32, V=50277, T=512, dtype="f32", penalties=True, bias="none",
             mask="row", sample=True),
        # greedy decoding of a large batch
        dict(nt, name="next_b256_greedy_bf16", B=256, V=50280, T=1024, dtype="bf16", penalties=True, bias="shared",
             mask="none", sample=False),
        # sampling for a large batch
        dict(nt, name="next_b256_sample_bf16", B=256, V=50280, T=1024, dtype="bf16", penalties=True, bias="none",
             mask="shared", sample=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    """Another case of the same ranges: 1 to 64 rows against weights of 200 to
    50,280 rows and 130 to 5,120 columns; 1 to 256 rows of 1,000 to 50,280
    logits with histories of 0 to 2,048 tokens."""
    op = rng.choice(["linear_w4", "process_logits", "next_tokens"])
    if op == "linear_w4":
        while True:
            M, N, K = _log_int(rng, 1, 64), _log_int(rng, 200, 50280), _log_int(rng, 130, 5120)
            if rng.random() < 0.5:
                K += -K % 64
            if N * K <= 50280 * 2560:
                break
        t = rng.choice(["f32", "bf16"])
        if t == "f32":
            M = min(M, 16)  # fp32 decoding is the small models' form
        return dict(op=op, M=M, N=N, K=K, G=rng.choice([32, 64, 128]), x=t, s=rng.choice([t, "f32"]),
                    zeros=rng.random() < 0.5)
    case = dict(op=op, B=_log_int(rng, 1, 256), V=_log_int(rng, 1000, 50280),
                T=0 if rng.random() < 0.2 else _log_int(rng, 1, 2048), dtype=rng.choice(["f32", "bf16"]),
                penalties=rng.random() < 0.7, bias=rng.choice(["none", "shared", "row"]),
                mask=rng.choice(["none", "shared", "row"]))
    if op == "next_tokens":
        case["sample"] = rng.random() < 0.5
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_w4(case, g) if case["op"] == "linear_w4" else _prepare_logits(case, g)


def _prepare_w4(c, g):
    N, K, G = c["N"], c["K"], c["G"]
    groups = -(-K // G)
    codes = torch.zeros(-(-N // 16), -(-K // 128), 16, 16, dtype=torch.int32, device="cuda")
    for shift in range(0, 32, 4):  # bell-shaped codes, as rounded weights have them
        q = torch.randn(codes.shape, generator=g, device="cuda").mul_(2.6).add_(8.0).round_().clamp_(0, 15)
        codes |= q.to(torch.int32) << shift
    x = torch.randn(c["M"], K, generator=g, device="cuda").to(TYPES[c["x"]])
    scales = ((0.5 + torch.rand(N, groups, generator=g, device="cuda")) * (0.4 / K ** 0.5)).to(TYPES[c["s"]])
    zeros = torch.randint(6, 11, (N, groups), generator=g, device="cuda", dtype=torch.uint8) if c["zeros"] else None
    return {"op": c["op"], "x": x, "codes": codes, "scales": scales, "zeros": zeros, "group_size": G}


def _prepare_logits(c, g):
    B, V, T = c["B"], c["V"], c["T"]
    rand = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    s = {"op": c["op"], "tokens": None, "lengths": None, "prompt_lengths": None, "repetition_penalty": None,
         "presence_penalty": None, "frequency_penalty": None, "bias": None, "allowed": None,
         "temperature": None, "seeds": None, "positions": None}
    s["logits"] = torch.randn(B, V, generator=g, device="cuda").mul_(3.0).to(TYPES[c["dtype"]])
    if T > 0:  # a skewed draw: frequent tokens repeat
        s["tokens"] = (rand(B, T).pow_(3.0) * V).long().clamp_(max=V - 1)
        s["lengths"] = ((rand(B) * T).long() + 1).clamp_(max=T)
        s["prompt_lengths"] = (rand(B) * s["lengths"] * 0.5).long()
    if c["penalties"]:
        s["repetition_penalty"] = 1.0 + 0.5 * rand(B)
        s["presence_penalty"] = rand(B)
        s["frequency_penalty"] = 0.5 * rand(B)
    if c["bias"] != "none":
        shape = (V,) if c["bias"] == "shared" else (B, V)
        s["bias"] = torch.randn(*shape, generator=g, device="cuda")
    if c["mask"] != "none":
        words = -(-V // 32)
        shape = (words,) if c["mask"] == "shared" else (B, words)
        bits = lambda: torch.randint(-2 ** 31, 2 ** 31, shape, generator=g, device="cuda", dtype=torch.int64)  # noqa: E731
        s["allowed"] = (bits() & bits()).to(torch.int32)  # a quarter of the vocabulary
    if c.get("sample"):
        s["temperature"] = 0.5 + rand(B)
        s["seeds"] = torch.randint(0, 2 ** 62, (B,), generator=g, device="cuda")
        s["positions"] = torch.randint(0, 2 ** 20, (B,), generator=g, device="cuda")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

ADJUST = ("tokens", "lengths", "prompt_lengths", "repetition_penalty", "presence_penalty", "frequency_penalty",
          "bias", "allowed")


def run(state):
    s = state
    if own:
        k = kernels()
        if s["op"] == "linear_w4":
            return k.linear_w4(s["x"], s["codes"], s["scales"], s["zeros"], group_size=s["group_size"])
        adjust = {name: s[name] for name in ADJUST}
        if s["op"] == "process_logits":
            return k.process_logits(s["logits"], **adjust)
        return k.next_tokens(s["logits"], **adjust, temperature=s["temperature"], seeds=s["seeds"],
                             positions=s["positions"])
    if s["op"] == "linear_w4":
        return _plain_w4(s["x"], s["codes"], s["scales"], s["zeros"], s["group_size"])
    z = _plain_adjusted(s)
    if s["op"] == "process_logits":
        return z.to(s["logits"].dtype)
    return _plain_choice(z, s["temperature"], s["seeds"], s["positions"])


def _plain_w4(x, codes, scales, zeros, group):
    M, K = x.shape
    N = scales.shape[0]
    shifts = torch.tensor(NIBBLE_SHIFTS, dtype=torch.int32, device=x.device)
    words = codes.unflatten(3, (4, 4)).permute(0, 2, 1, 4, 3)  # [rows / 16][row][columns / 128][j][t]
    w = ((words.unsqueeze(-1) >> shifts) & 15).flatten(0, 1).flatten(1)[:N, :K].float()
    at = torch.arange(K, device=x.device) // group
    w = w - (8.0 if zeros is None else zeros.float()[:, at])
    w = w * scales.float()[:, at]
    return (x.float() @ w.t()).to(x.dtype)


def _plain_adjusted(s):
    z = s["logits"].float()
    B, V = z.shape
    if s["tokens"] is not None and s["repetition_penalty"] is not None:
        tokens = s["tokens"]
        at = torch.arange(tokens.shape[1], device=z.device)
        inside = at < s["lengths"][:, None]
        generated = inside & (at >= s["prompt_lengths"][:, None])
        seen = torch.zeros_like(z).scatter_add_(1, tokens, inside.float()) > 0
        count = torch.zeros_like(z).scatter_add_(1, tokens, generated.float())
        r = s["repetition_penalty"][:, None]
        z = torch.where(seen, torch.where(z > 0, z / r, z * r), z)
        z = z - s["frequency_penalty"][:, None] * count
        z = z - s["presence_penalty"][:, None] * (count > 0)
    if s["bias"] is not None:
        z = z + s["bias"]
    if s["allowed"] is not None:
        bit = torch.arange(32, dtype=torch.int32, device=z.device)
        ok = ((s["allowed"].unsqueeze(-1) >> bit) & 1).flatten(-2)[..., :V] != 0
        z = torch.where(ok, z, float("-inf"))
    return z


def _mul_hi_lo(a, m):
    """High and low 32 bits of a * m, both below 2^32, in int64."""
    p = a * m  # wraps modulo 2^64: the bits are those of the product
    return (p >> 32) & 0xFFFFFFFF, p & 0xFFFFFFFF


def _plain_noise(seeds, positions, V):
    """-log(-log u) of row b, token i in 64 bits: u in (0, 1) from word i % 4
    of the generator's block i / 4 at the row's seed and position."""
    B, n = seeds.shape[0], -(-V // 4)
    c0 = torch.arange(n, device=seeds.device).expand(B, n)
    c1 = (positions & 0xFFFFFFFF)[:, None].expand(B, n)
    c2 = ((positions >> 32) & 0xFFFFFFFF)[:, None].expand(B, n)
    c3 = torch.zeros_like(c0)
    k0, k1 = (seeds & 0xFFFFFFFF)[:, None], ((seeds >> 32) & 0xFFFFFFFF)[:, None]
    for _ in range(PHILOX_ROUNDS):
        h0, l0 = _mul_hi_lo(c0, PHILOX_M[0])
        h1, l1 = _mul_hi_lo(c2, PHILOX_M[1])
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + PHILOX_W[0]) & 0xFFFFFFFF, (k1 + PHILOX_W[1]) & 0xFFFFFFFF
    bits = torch.stack((c0, c1, c2, c3), dim=-1).reshape(B, -1)[:, :V]
    v = (bits.double() + 0.5) * 2.0 ** -32  # u = 1 - v
    return -torch.log(-torch.log1p(-v))


def _plain_choice(z, temperature, seeds, positions):
    if temperature is None:
        ids, scaled = z.argmax(dim=-1), z
    else:
        scaled = z / temperature[:, None]
        score = z.double() / temperature.double()[:, None] + _plain_noise(seeds, positions, z.shape[1])
        ids = score.argmax(dim=-1)
    chosen = scaled.gather(1, ids[:, None])[:, 0]
    top = scaled.max(dim=-1).values
    total = torch.exp(scaled - top[:, None]).sum(dim=-1)
    logprob = torch.where(top == float("-inf"), top, chosen - top - torch.log(total))
    return ids, logprob


# ---------------------------------------------------------------------------
# bytes and operations of one pass
# ---------------------------------------------------------------------------

def work(case):
    c = case
    size = {"f32": 4, "bf16": 2}
    if c["op"] == "linear_w4":
        M, N, K = c["M"], c["N"], c["K"]
        groups = -(-K // c["G"])
        nbytes = N * K / 2 + N * groups * (size[c["s"]] + (1 if c["zeros"] else 0)) + (M * K + M * N) * size[c["x"]]
        return {"bytes": nbytes, "flops": 2.0 * M * N * K}
    B, V, T = c["B"], c["V"], c["T"]
    sample = c.get("sample", False)
    nbytes = B * V * size[c["dtype"]] * (2 if c["op"] == "process_logits" else 1)
    if T > 0 and c["penalties"]:
        nbytes += B * T / 2 * 8 + B * 28  # half of each history is in use, on average
    nbytes += {"none": 0, "shared": V * 4, "row": B * V * 4}[c["bias"]]
    nbytes += {"none": 0, "shared": V / 8, "row": B * V / 8}[c["mask"]]
    if c["op"] == "next_tokens":
        nbytes += B * 12 + (B * 20 if sample else 0)
    per = 4 * c["penalties"] + (c["bias"] != "none") + (0 if c["op"] == "process_logits" else 4 + 60 * sample)
    return {"bytes": nbytes, "flops": float(max(1, per) * B * V)}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear_w4":
        return _exact_w4(case, s)
    return _exact_logits(case, s)


def _exact_w4(c, s):
    """Each column fetched from its word and bit, products summed in 64 bits."""
    N, K, G = c["N"], c["K"], c["G"]
    x = s["x"].double()
    y = torch.empty(c["M"], N, dtype=torch.float64, device="cuda")
    # (word, bit) of column k in a row of 16 words a block
    k = np.arange(K)
    tile, inner = k // 128, k % 128
    word = tile * 16 + 4 * ((inner % 32) // 8) + inner // 32
    bit = 4 * ((inner % 8) // 2) + 16 * (inner % 2)
    word_t, bit_t = torch.from_numpy(word).cuda(), torch.from_numpy(bit).cuda()
    words = s["codes"].transpose(1, 2).reshape(-1, (K + 127) // 128 * 16)
    rows = max(1, (1 << 24) // K)
    for n0 in range(0, N, rows):
        part = slice(n0, min(N, n0 + rows))
        code = (words[part].long()[:, word_t] >> bit_t) % 16
        w = code.double()
        for g0 in range(0, K, G):
            cols, grp = slice(g0, min(K, g0 + G)), g0 // G
            zero = 8.0 if s["zeros"] is None else s["zeros"][part, grp, None].double()
            w[:, cols] = (w[:, cols] - zero) * s["scales"][part, grp, None].double()
        y[:, part] = torch.einsum("mk,nk->mn", x, w)
    return y


def _exact_noise(seed, position, V):
    """Row noise in numpy, 32-bit words held in uint64."""
    mask = np.uint64(0xFFFFFFFF)
    n = -(-V // 4)
    c = [np.arange(n, dtype=np.uint64), np.full(n, position & 0xFFFFFFFF, np.uint64),
         np.full(n, (position >> 32) & 0xFFFFFFFF, np.uint64), np.zeros(n, np.uint64)]
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for r in range(PHILOX_ROUNDS):
        a, b = c[0] * np.uint64(PHILOX_M[0]), c[2] * np.uint64(PHILOX_M[1])
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(key[0]), b & mask,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(key[1]), a & mask]
        key = [(key[0] + PHILOX_W[0]) % 2 ** 32, (key[1] + PHILOX_W[1]) % 2 ** 32]
    word = np.stack(c, axis=1).reshape(-1)[:V].astype(np.float64)
    v = (word + 0.5) / 2.0 ** 32
    return -np.log(-np.log1p(-v))


def _exact_logits(c, s):
    """Row by row in numpy."""
    host = {k: (v.float() if v.dtype == torch.bfloat16 else v).cpu().numpy() if isinstance(v, torch.Tensor) else v
            for k, v in s.items()}
    B, V = c["B"], c["V"]
    ids, logprobs = np.zeros(B, np.int64), np.zeros(B)
    out = np.zeros((B, V)) if c["op"] == "process_logits" else None
    for b in range(B):
        z = host["logits"][b].astype(np.float64)
        if host["tokens"] is not None and c["penalties"]:
            n, p = int(host["lengths"][b]), int(host["prompt_lengths"][b])
            history = host["tokens"][b, :n]
            count = np.bincount(history[p:], minlength=V).astype(np.float64)
            seen = np.unique(history)
            r = float(host["repetition_penalty"][b])
            z[seen] = np.where(z[seen] > 0, z[seen] / r, z[seen] * r)
            z -= float(host["frequency_penalty"][b]) * count
            z[count > 0] -= float(host["presence_penalty"][b])
        if host["bias"] is not None:
            z += host["bias"] if host["bias"].ndim == 1 else host["bias"][b]
        if host["allowed"] is not None:
            words = host["allowed"] if host["allowed"].ndim == 1 else host["allowed"][b]
            bits = np.unpackbits(np.ascontiguousarray(words).view(np.uint8), bitorder="little")[:V]
            z[bits == 0] = -np.inf
        if out is not None:
            out[b] = z
            continue
        t = float(host["temperature"][b]) if host["temperature"] is not None else 1.0
        zt = z / t
        score = zt + _exact_noise(int(host["seeds"][b]), int(host["positions"][b]), V) if c["sample"] else zt
        ids[b] = int(np.argmax(score))
        top = zt.max()
        logprobs[b] = top if np.isneginf(top) else zt[ids[b]] - top - np.log(np.exp(zt - top).sum())
    if out is not None:
        return out
    return ids, logprobs
