"""The operators of a transformer on encrypted data: cases, inputs, the plain form of each operator and its value in 64 bits.

Everything lies in RNS-CKKS form: a ciphertext is two polynomials, a polynomial is one residue vector (N words, NTT domain) per prime of
its level.  Feature i of a token matrix is one ciphertext; tokens (or the sequences of a batch) lie in its slots, further tokens in further
rows.  Uniform residues are what encryption makes of any message, so the inputs are uniform residues.

  linear    y[r][j] = tok[r] * mul[j] * sum_i w[j][i] x[r][i]            int8 weights; one integer per channel, one plaintext per row of tokens
  angles    cos, sin of pos[axis[i]][t] * freq[i]                        the messages of rotary positions with several axes (time, height, width)
  rope      (x0, x1) -> (x0 C - x1 S, x0 S + x1 C)                       the rotation of the pairs (i, i + dim/2), C and S the encoded messages
  scores    P[h][t][s]  = sum_a q[t][h][a] (x) k[s][h'][a]               linear attention with a decay per head, in chunks; (x) is the product of
  out       O[h][t][b]  = g[h][t] sum_a q[t][h][a] (x) S[h][a][b]          two ciphertexts before relinearisation (three polynomials), the chunk's
                          + sum_s d[h][t-s] P[h][t][s] (x) v[s][h'][b]     own part causal (s <= t); h' = the head of keys and values that head h shares
  state     S'[h][a][b] = g[h] S[h][a][b] + sum_s d[h][n-1-s] k[s][h'][a] (x) v[s][h'][b]       one token: the recurrent form
"""
import functools
import itertools
import math

import numpy as np
import torch

own = False

DEVICE = torch.device("cuda" if torch.cuda.is_available() else "cpu")

# Parameter sets (ring degree N, q primes L, bits of the first and of the scaling primes, dnum) of the repository's own configurations and tests:
# the key-switch benchmark's 60 / 56-bit chain, the generated networks' 51 / 50-bit chain, the small rings of the parity tests.
SETS = {
    1024: (7, 60, 51, 3),
    2048: (10, 60, 55, 3),
    4096: (6, 60, 50, 3),
    8192: (4, 60, 50, 2),
    16384: (4, 60, 56, 2),
    32768: (6, 51, 50, 3),
    65536: (25, 60, 56, 4),
}


def _linear(N, level, rows, n_in, n_out, mul, tok):
    return {"op": "linear", "N": N, "level": level, "rows": rows, "n_in": n_in, "n_out": n_out, "mul": mul, "tok": tok}


def _angles(slots, pairs, axes):
    return {"op": "angles", "N": 2 * slots, "level": 1, "slots": slots, "pairs": pairs, "axes": axes}


def _rope(N, level, heads, rows, dim):
    return {"op": "rope", "N": N, "level": level, "heads": heads, "rows": rows, "dim": dim}


def _scores(N, level, heads, kv, tokens, dim):
    return {"op": "scores", "N": N, "level": level, "heads": heads, "kv": kv, "tokens": tokens, "dk": dim}


def _out(N, level, heads, kv, tokens, dk, dv, chunk):
    return {"op": "out", "N": N, "level": level, "heads": heads, "kv": kv, "tokens": tokens, "dk": dk, "dv": dv, "chunk": chunk}


def _state(N, level, heads, kv, tokens, dk, dv):
    return {"op": "state", "N": N, "level": level, "heads": heads, "kv": kv, "tokens": tokens, "dk": dk, "dv": dv}


def listed():
    return [
        # a classifier's last layer on the smallest ring of the tests: latency
        dict(_linear(1024, 2, 1, 16, 10, False, False), name="linear_head"),
        # a projection with odd sizes, three rows of tokens, both scales
        dict(_linear(4096, 3, 3, 333, 77, True, True), name="linear_ragged"),
        # an ordinary hidden layer
        dict(_linear(8192, 4, 1, 512, 512, True, False), name="linear_hidden"),
        # the joint projection to queries, keys and values of a wide layer: the largest product
        dict(_linear(16384, 3, 1, 768, 2304, True, True), name="linear_qkv"),
        # positions of a long video, all slots of the largest ring, three axes
        dict(_angles(32768, 64, 3), name="angles_video"),
        # one small head: latency
        dict(_rope(1024, 2, 1, 1, 8), name="rope_small"),
        # all heads of a layer, the tables shared by the heads
        dict(_rope(16384, 4, 16, 1, 64), name="rope_layer"),
        # a decoding step: the state takes one token in (recurrent form)
        dict(_state(8192, 4, 4, 4, 1, 32, 32), name="state_token"),
        # a decoding step of a small model: one token reads the state
        dict(_out(1024, 2, 2, 2, 1, 32, 32, False), name="out_token"),
        # a prompt's chunk: scores, four heads sharing two heads of keys
        dict(_scores(4096, 3, 4, 2, 32, 32), name="scores_chunk"),
        # a prompt's chunk: the state's part and the chunk's own part
        dict(_out(8192, 3, 2, 1, 16, 24, 32, True), name="out_chunk"),
        # a prompt's chunk goes into the state, odd sizes
        dict(_state(2048, 3, 3, 1, 19, 21, 33), name="state_chunk"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = {w: max(work(c)[w] for c in listed()) for w in ("bytes", "flops")}
    while True:
        N = rng.choice([1024, 2048, 4096, 8192, 16384, 32768])
        level = rng.randint(1, min(5, SETS[N][0]))
        heads = rng.choice([1, 2, 3, 4, 6, 8])
        kv = rng.choice([k for k in (1, 2, 3, 4, 6, 8) if heads % k == 0])
        c = rng.choice([
            lambda: _linear(N, level, rng.choice([1, 1, 2, 3, 5]), _spread(rng, 8, 1536), _spread(rng, 8, 1536), rng.random() < 0.6, rng.random() < 0.5),
            lambda: _linear(N, level, rng.choice([1, 1, 2, 3, 5]), _spread(rng, 8, 1536), _spread(rng, 8, 1536), rng.random() < 0.6, rng.random() < 0.5),
            lambda: _angles(_spread(rng, 400, 32768), _spread(rng, 4, 96), rng.randint(1, 3)),
            lambda: _rope(N, level, _spread(rng, 1, 16), rng.choice([1, 1, 2, 3]), 2 * _spread(rng, 4, 64)),
            lambda: _scores(N, level, heads, kv, _spread(rng, 2, 48), _spread(rng, 4, 64)),
            lambda: _out(N, level, heads, kv, _spread(rng, 1, 32), _spread(rng, 4, 48), _spread(rng, 4, 48), rng.random() < 0.6),
            lambda: _state(N, level, heads, kv, _spread(rng, 1, 32), _spread(rng, 4, 48), _spread(rng, 4, 48)),
        ])()
        if c["op"] == "angles":
            c["N"] = 2 * c["slots"]
        w = work(c)
        if w["bytes"] <= 0.6 * most["bytes"] and w["flops"] <= most["flops"] and _products(c) <= max(map(_products, listed())):
            return c


def _products(case):
    """products of two ciphertexts, in words: what the plain form of the attention operators spends its time on"""
    if case["op"] not in ("scores", "out", "state"):
        return 0
    heads, n, dk, dv = case["heads"], case["tokens"], case["dk"], case.get("dv", 0)
    terms = {"scores": n * n * dk, "out": n * dv * (dk + n * case.get("chunk", 0)), "state": n * dk * dv}[case["op"]]
    return heads * terms * case["level"] * case["N"]


# ---- the prime chain of a parameter set -----------------------------------------------------------------------------------------------
def _prime(n):
    if n < 41:
        return n in (2, 3, 5, 7, 11, 13, 17, 19, 23, 29, 31, 37)
    s = ((n - 1) & (1 - n)).bit_length() - 1
    return all(n % b and (pow(b, (n - 1) >> s, n) == 1 or any(pow(b, (n - 1) >> r, n) == n - 1 for r in range(1, s + 1)))
               for b in (2, 3, 5, 7, 11, 13, 17, 19, 23, 29, 31, 37))


def _walk(start, step):
    return next(c for c in itertools.count(start + step, step) if _prime(c))


@functools.lru_cache(None)
def _primes(N):
    """q primes of the parameter set: the last one the first above 2^sf, then alternately below and above it (the step up skips one
    candidate), the first prime the one before the first above 2^q0."""
    L, q0, sf, _ = SETS[N]
    step = 2 * N
    anchor = _walk((1 << sf) + 1, step)
    below = itertools.accumulate(itertools.repeat(-step), _walk, initial=anchor)
    above = itertools.accumulate(itertools.repeat(step), lambda c, s: _walk(c + s, s), initial=anchor)
    next(below), next(above)
    chain = [next(above if i % 2 else below) for i in range(L - 2)]
    return [_walk(_walk((1 << q0) + 1, step), -step)] + chain[::-1] + [anchor]


# ---- inputs ---------------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    N, level = c["N"], c["level"]
    st = {"case": c}

    def uniform(*shape):
        return torch.randint(0, 1 << 62, (*shape, level, N), generator=g, device=DEVICE) % st["q"]

    def zeros(*shape):
        return torch.zeros(*shape, level, N, dtype=torch.int64, device=DEVICE)

    if c["op"] == "angles":
        # frequencies of the usual ladder, pairs dealt to the axes in turn; a video's patches in raster order, starting far into it
        n = c["slots"]
        t = torch.arange(n, device=DEVICE, dtype=torch.float64)
        side = max(1, math.isqrt(n // 8))
        first = torch.randint(0, 1 << 20, (1,), generator=g, device=DEVICE).double()
        st["pos"] = torch.stack([first + t // (side * side), t // side % side, t % side])[: c["axes"]].contiguous()
        st["freq"] = [10000.0 ** (-i / c["pairs"]) for i in range(c["pairs"])]
        st["axis"] = [i % c["axes"] for i in range(c["pairs"])]
        st["cos"], st["sin"] = (torch.zeros(c["pairs"], n, dtype=torch.float64, device=DEVICE) for _ in range(2))
    else:
        st["q"] = torch.tensor(_primes(N)[:level], device=DEVICE).view(level, 1)
        sf = SETS[N][2]
    if c["op"] == "linear":
        st["x"] = uniform(c["rows"], c["n_in"], 2)
        st["w"] = (torch.randn(c["n_out"], c["n_in"], generator=g, device=DEVICE) * 40).round().clamp(-127, 127).to(torch.int8)
        # the channel's scale times the scaling factor, as an integer; the row's scales as an encoded plaintext
        st["mul"] = (torch.rand(c["n_out"], generator=g, device=DEVICE, dtype=torch.float64) * 0.02 * 2.0**sf).round().long() if c["mul"] else None
        st["tok"] = uniform(c["rows"]) if c["tok"] else None
        st["y"] = zeros(c["rows"], c["n_out"], 2)
    if c["op"] == "rope":
        st["x"] = uniform(c["heads"], c["rows"], c["dim"], 2)
        st["cos"], st["sin"] = uniform(c["rows"], c["dim"] // 2), uniform(c["rows"], c["dim"] // 2)
        st["y"] = zeros(c["heads"], c["rows"], c["dim"], 2)
    if c["op"] in ("scores", "out", "state"):
        H, n = c["heads"], c["tokens"]
        # decay of head h: 1 - 2^-(5 + h), in powers of the distance, times the scaling factor
        rate = 1 - 2.0 ** -(5 + torch.arange(H, device=DEVICE, dtype=torch.float64))
        power = (rate[:, None] ** torch.arange(n + 1, device=DEVICE, dtype=torch.float64) * 2.0**sf).round().long()
        st["decay"], st["grown"], st["keep"] = power[:, :n].contiguous(), power[:, 1:].contiguous(), power[:, n].contiguous()
        if c["op"] != "state":
            st["query"] = uniform(n, H, c["dk"], 2)
        if c["op"] != "out":
            st["k"] = uniform(n, c["kv"], c["dk"], 2)
        if c["op"] != "scores":
            st["S"] = uniform(H, c["dk"], c["dv"], 2)
        if c["op"] == "state" or c.get("chunk"):
            st["v"] = uniform(n, c["kv"], c["dv"], 2)
        if c.get("chunk"):
            st["P"] = uniform(H, n, n, 2)
        st["y"] = zeros(H, *{"scores": (n, n), "out": (n, c.get("dv")), "state": (c["dk"], c.get("dv"))}[c["op"]], 3)
    if own:  # the handle that a program keeps: the context of its parameter set, and the stream that it works on -- one for a context, whose
        # calls may share its workspace and follow each other
        st["rt"] = _context(1024 if c["op"] == "angles" else N)
        st["stream"] = _stream(1024 if c["op"] == "angles" else N)
        torch.cuda.synchronize()
    return st


@functools.lru_cache(None)
def _context(N):
    import ace_compiler_amd as A

    rt = A.AceHip(N, *SETS[N])
    assert rt.primes[: rt.L] == _primes(N)
    return rt


@functools.lru_cache(None)
def _stream(N):
    return torch.cuda.Stream()


# ---- one pass -------------------------------------------------------------------------------------------------------------------------
def run(st):
    return _RUN[st["case"]["op"], bool(own)](st)


def _mulc(a, c, q):
    """a * c mod q for a, q < 2^61, 0 <= c < 2^31: the quotient, below 2^31, from a product in 64 bits of floating point is at most one off"""
    r = a * c - torch.floor(a.double() * c / q).long() * q
    r = torch.where(r < 0, r + q, r)
    return torch.where(r >= q, r - q, r)


def _mul(a, b, q):
    """a * b mod q for a, b < q: by the halves of b"""
    return (_mulc(_mulc(a, b >> 30, q), 1 << 30, q) + _mulc(a, b & ((1 << 30) - 1), q)) % q


def _linear_plain(st):
    x, w, q = st["x"], st["w"].double(), st["q"]
    rows, n_in = x.shape[:2]
    # sums of at most 2^12 products of 2^7 by 2^31: exact in 64 bits of floating point
    low, high = ((w @ part.double().view(rows, n_in, -1)).view(rows, -1, *x.shape[2:]).long() for part in (x & ((1 << 31) - 1), x >> 31))
    y = (_mulc(high % q, 1 << 30, q) * 2 + low) % q
    if st["mul"] is not None:
        y = _mul(y, st["mul"].view(-1, 1, 1, 1) % q, q)
    if st["tok"] is not None:
        y = _mul(y, st["tok"][:, None, None], q)
    return y


def _linear_own(st):
    c, x, y = st["case"], st["x"], st["y"]
    st["rt"].linear_i8(_mat(st, y, "row col comp"), _mat(st, x, "row col comp"), st["w"].data_ptr(), c["n_in"], c["rows"], c["n_in"], c["n_out"], 2, c["level"],
                       d_mul=st["mul"].data_ptr() if c["mul"] else 0, d_tok=st["tok"].data_ptr() if c["tok"] else 0, tok_stride=c["level"] * c["N"],
                       stream=st["stream"].cuda_stream)
    return y


def _angles_plain(st):
    angle = st["pos"][st["axis"]] * torch.tensor(st["freq"], dtype=torch.float64, device=DEVICE)[:, None]
    return {"cos": torch.cos(angle), "sin": torch.sin(angle)}


def _angles_own(st):
    n = st["case"]["slots"]
    st["rt"].rope_messages(st["cos"].data_ptr(), st["sin"].data_ptr(), n, st["pos"].data_ptr(), n, n, st["freq"], st["axis"], st["case"]["axes"],
                           stream=st["stream"].cuda_stream)
    return {"cos": st["cos"], "sin": st["sin"]}


def _rope_plain(st):
    q, C, S = st["q"], st["cos"][None, :, :, None], st["sin"][None, :, :, None]
    x0, x1 = st["x"].chunk(2, dim=2)
    return torch.cat([(_mul(x0, C, q) + q - _mul(x1, S, q)) % q, (_mul(x0, S, q) + _mul(x1, C, q)) % q], dim=2)


def _rope_own(st):
    c, x, y = st["case"], st["x"], st["y"]
    words = c["level"] * c["N"]
    st["rt"].rope(_mat(st, y, "head row col comp"), _mat(st, x, "head row col comp"), st["cos"].data_ptr(), st["sin"].data_ptr(), words, words * (c["dim"] // 2),
                  c["heads"], c["rows"], c["dim"], 2, c["level"], stream=st["stream"].cuda_stream)
    return y


def _dot(a, b, q):
    """Products of matrices of residues: [limb][N][h][m][k] by [limb][N][h][k][n], mod q ([limb][1][1][1][1]).  In thirds of 20 bits: sums of at most
    2^11 products below 2^40 are exact in 64 bits of floating point, three of them below 2^53."""
    third = lambda x: [(x >> s & ((1 << 20) - 1)).double() for s in (0, 20, 40)]
    A, B = third(a), third(b)
    part = [sum(A[i] @ B[s - i] for i in range(3) if 0 <= s - i < 3).long() for s in range(5)]
    return functools.reduce(lambda r, p: (_mulc(r, 1 << 20, q) + p) % q, part[-2::-1], part[-1] % q)


def _points(x, h, m, k):
    """axes h, m, k of [.., 2, limb, N] as [limb][N][h][m][k] for each of the two polynomials"""
    return [x.select(3, p).permute(3, 4, h, m, k) for p in (0, 1)]


def _product(a, b, q):
    """the three polynomials of the product of two matrices of ciphertexts, as [h][m][n][3][limb][N]"""
    (a0, a1), (b0, b1) = a, b
    y = [_dot(a0, b0, q), _dot(torch.cat([a0, a1], -1), torch.cat([b1, b0], -2), q), _dot(a1, b1, q)]
    return torch.stack(y, -1).permute(2, 3, 4, 5, 0, 1)


def _shared(x, st):
    """keys or values [token][kv][d] for each of the heads that share them"""
    return x.repeat_interleave(st["case"]["heads"] // st["case"]["kv"], dim=1)


def _scores_plain(st):
    q, n = st["q"], st["case"]["tokens"]
    y = _product(_points(st["query"], 1, 0, 2), _points(_shared(st["k"], st), 1, 2, 0), q.view(-1, 1, 1, 1, 1))
    return torch.where(torch.ones(n, n, dtype=torch.bool, device=DEVICE).tril()[..., None, None, None], y, 0)


def _scores_own(st):
    c = st["case"]
    st["rt"].linattn_scores(_mat(st, st["y"], "head row col comp"), _mat(st, st["query"], "row head col comp"), _mat(st, st["k"], "row head col comp"), c["heads"], c["kv"],
                            c["tokens"], c["tokens"], c["dk"], c["level"], causal=True, stream=st["stream"].cuda_stream)
    return st["y"]


def _out_plain(st):
    q, n = st["q"], st["case"]["tokens"]
    q5 = q.view(-1, 1, 1, 1, 1)
    query = _mul(st["query"], st["grown"].T[:, :, None, None, None, None] % q, q) if st["case"]["chunk"] else st["query"]
    y = _product(_points(query, 1, 0, 2), _points(st["S"], 0, 1, 2), q5)
    if st["case"]["chunk"]:
        t = torch.arange(n, device=DEVICE)
        d = torch.where(t[:, None] >= t, st["decay"][:, (t[:, None] - t).clamp(min=0)], 0)[..., None, None, None]
        y = (y + _product(_points(_mul(st["P"], d % q, q), 0, 1, 2), _points(_shared(st["v"], st), 1, 0, 2), q5)) % q
    return y


def _out_own(st):
    c, chunk = st["case"], st["case"]["chunk"]
    st["rt"].linattn_out(_mat(st, st["y"], "head row col comp"), _mat(st, st["query"], "row head col comp"), _mat(st, st["S"], "head row col comp"),
                         _mat(st, st["P"], "head row col comp") if chunk else None, _mat(st, st["v"], "row head col comp") if chunk else None,
                         c["heads"], c["kv"], c["tokens"], c["tokens"] if chunk else 0, c["dk"], c["dv"], c["level"], d_in=st["grown"].data_ptr() if chunk else 0,
                         d_decay=st["decay"].data_ptr() if chunk else 0, causal=True, stream=st["stream"].cuda_stream)
    return st["y"]


def _state_plain(st):
    q, n = st["q"], st["case"]["tokens"]
    k = _shared(st["k"], st)
    if n > 1:
        k = _mul(k, st["decay"].flip(1).T[:, :, None, None, None, None] % q, q)
    y = _product(_points(k, 1, 2, 0), _points(_shared(st["v"], st), 1, 0, 2), q.view(-1, 1, 1, 1, 1))
    kept = _mul(st["S"], st["keep"][:, None, None, None, None, None] % q, q)
    return torch.cat([(y[:, :, :, :2] + kept) % q, y[:, :, :, 2:]], dim=3)


def _state_own(st):
    c = st["case"]
    st["rt"].linattn_state(_mat(st, st["y"], "head row col comp"), _mat(st, st["S"], "head row col comp"), _mat(st, st["k"], "row head col comp"),
                           _mat(st, st["v"], "row head col comp"), c["heads"], c["kv"], c["tokens"], c["dk"], c["dv"], c["level"], d_keep=st["keep"].data_ptr(),
                           d_decay=st["decay"].data_ptr() if c["tokens"] > 1 else 0, stream=st["stream"].cuda_stream)
    return st["y"]


def _mat(st, t, axes):
    """the framework's view of a tensor of ciphertexts whose leading axes are named"""
    return st["rt"].mat(t.data_ptr(), **dict(zip(axes.split(), t.stride())))


_RUN = {
    ("linear", False): _linear_plain, ("angles", False): _angles_plain, ("rope", False): _rope_plain,
    ("scores", False): _scores_plain, ("out", False): _out_plain, ("state", False): _state_plain,
    ("linear", True): _linear_own, ("angles", True): _angles_own, ("rope", True): _rope_own,
    ("scores", True): _scores_own, ("out", True): _out_own, ("state", True): _state_own,
}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------------------
def work(case):
    """bytes: every input read once, every output written once.  flops: two for each term of a sum; a product of a word by an int8 weight is
    taken as one, a product of two words as one, an angle's cosine and sine as one each."""
    c = case
    limb = 8 * c["N"] * c["level"]
    if c["op"] == "linear":
        words = c["rows"] * (2 * (c["n_in"] + c["n_out"]) + c["tok"])
        return {"bytes": words * limb + c["n_in"] * c["n_out"] + 8 * c["n_out"] * c["mul"], "flops": 2 * c["rows"] * c["n_in"] * c["n_out"] * 2 * limb // 8}
    if c["op"] == "angles":
        return {"bytes": 8 * c["slots"] * (2 * c["pairs"] + c["axes"]), "flops": 3 * c["slots"] * c["pairs"]}
    if c["op"] == "rope":
        return {"bytes": limb * c["rows"] * c["dim"] * (4 * c["heads"] + 1), "flops": 2 * limb // 8 * c["heads"] * c["rows"] * c["dim"] * 4}
    H, kv, n, dk, dv = c["heads"], c["kv"], c["tokens"], c["dk"], c.get("dv", 0)
    seen = n * (n + 1) // 2
    if c["op"] == "scores":
        return {"bytes": limb * (2 * n * dk * (H + kv) + 3 * H * seen), "flops": 2 * 4 * H * seen * dk * limb // 8}
    if c["op"] == "out":
        polys = 2 * H * n * dk + 2 * H * dk * dv + 3 * H * n * dv + (2 * H * seen + 2 * n * kv * dv if c["chunk"] else 0)
        return {"bytes": limb * polys, "flops": 2 * 4 * H * dv * (n * dk + seen * c["chunk"]) * limb // 8}
    return {"bytes": limb * (2 * n * kv * (dk + dv) + 5 * H * dk * dv), "flops": 2 * 4 * H * dk * dv * n * limb // 8}


# ---- the operators' values from their definitions, with whole numbers of any length (angles: in extended floating point) -----------------
def exact(case, seed):
    c = case
    if c["op"] == "angles":
        if c["slots"] * c["pairs"] > 1 << 22:
            return None
        st = prepare(case, seed)
        angle = st["pos"].cpu().numpy()[st["axis"]] * np.array(st["freq"])[:, None]
        return {"cos": np.cos(angle.astype(np.longdouble)).astype(np.float64), "sin": np.sin(angle.astype(np.longdouble)).astype(np.float64)}
    terms = {"linear": lambda: c["rows"] * c["n_in"] * c["n_out"] * 2 * c["level"] * c["N"], "rope": lambda: 8 * c["heads"] * c["rows"] * c["dim"] * c["level"] * c["N"]}
    if terms.get(c["op"], lambda: 4 * _products(c))() > 1 << 25:
        return None
    st = prepare(case, seed)
    big = {k: v.cpu().numpy().astype(object) for k, v in st.items() if isinstance(v, torch.Tensor)}
    q = big["q"]
    if c["op"] == "linear":
        y = np.tensordot(big["w"], big["x"], (1, 1)).swapaxes(0, 1)
        y = y * (big["mul"][:, None, None, None] if c["mul"] else 1) * (big["tok"][:, None, None] if c["tok"] else 1) % q
    elif c["op"] == "rope":
        half = c["dim"] // 2
        y = np.zeros_like(big["x"])
        for i in range(half):
            C, S = big["cos"][None, :, i, None], big["sin"][None, :, i, None]
            a, b = big["x"][:, :, i], big["x"][:, :, i + half]
            y[:, :, i], y[:, :, i + half] = (a * C - b * S) % q, (a * S + b * C) % q
    else:
        y = np.zeros(st["y"].shape, dtype=object)
        H, n, group = c["heads"], c["tokens"], c["heads"] // c["kv"]
        pair = lambda a, b: np.stack([a[0] * b[0], a[0] * b[1] + a[1] * b[0], a[1] * b[1]])
        for h, i, j in itertools.product(*(range(s) for s in st["y"].shape[:3])):
            kv = h // group
            if c["op"] == "scores" and j <= i:
                y[h, i, j] = sum(pair(big["query"][i, h, a], big["k"][j, kv, a]) for a in range(c["dk"])) % q
            elif c["op"] == "out":
                g = big["grown"][h, i] if c["chunk"] else 1
                y[h, i, j] = sum(g * pair(big["query"][i, h, a], big["S"][h, a, j]) for a in range(c["dk"])) % q
                if c["chunk"]:
                    y[h, i, j] = (y[h, i, j] + sum(big["decay"][h, i - s] * pair(big["P"][h, i, s], big["v"][s, kv, j]) for s in range(i + 1))) % q
            elif c["op"] == "state":
                y[h, i, j] = sum((big["decay"][h, n - 1 - s] if n > 1 else 1) * pair(big["k"][s, kv, i], big["v"][s, kv, j]) for s in range(n))
                y[h, i, j, :2] += big["keep"][h] * big["S"][h, i, j]
                y[h, i, j] %= q
    return y.astype(np.int64)
