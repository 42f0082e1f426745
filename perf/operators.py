"""The operators on 8-bit rows as cases: writing rows into a store, reading them back, products of two stores' rows,
and the distance of every row to the nearest of many centres.

A store keeps every row as e4m3 codes with one power-of-two scale per 128 elements.  Its arrays:
``codes`` float8_e4m3fn [capacity, pitch] (pitch = dim rounded up to 16, padding codes 0), ``scales`` uint8
[tiles of 128 rows, words, 32, 4, 4] (biased exponent of block 4 w + i of row 128 t + 32 j + r at [t, w, r, j, i]) and
``norms`` float32 [capacity], the squared norm of each row as stored.
"""
import torch

own = False

BLOCK = 128
LOW, BIAS = -117, 127
SIZES = {"float32": 4, "float16": 2, "bfloat16": 2}


def listed():
    return [
        # one new embedding added to a store of the small configuration (20 000 x 64): latency
        {"name": "write_1x64_f32", "op": "write", "n": 1, "dim": 64, "dtype": "float32", "capacity": 20000, "start": 19333},
        # a batch of embeddings as a model hands them over, behind what the store holds already
        {"name": "write_4096x1024_bf16", "op": "write", "n": 4096, "dim": 1024, "dtype": "bfloat16", "capacity": 40000, "start": 30001},
        # an odd width and an odd number of half rows
        {"name": "write_100003x50_f16", "op": "write", "n": 100003, "dim": 50, "dtype": "float16", "capacity": 100003, "start": 0},
        # a block of a large float32 matrix on its way into 8 bits
        {"name": "write_2000000x256_f32", "op": "write", "n": 2000000, "dim": 256, "dtype": "float32", "capacity": 2000000, "start": 0},
        # the 512 selected rows of the small configuration, read back for use
        {"name": "read_512_of_20000x64_f32", "op": "read", "m": 512, "n": 20000, "dim": 64, "dtype": "float32"},
        # all rows of a wide store as half precision, for a path that reads a matrix
        {"name": "read_1000000x1024_f16", "op": "read", "m": 0, "n": 1000000, "dim": 1024, "dtype": "float16"},
        # one new row against a whole store: the bytes of the store
        {"name": "products_1x1000000x256_f32", "op": "products", "n": 1, "k": 1000000, "dim": 256, "dtype": "float32"},
        # a ragged block of similarities of an odd width
        {"name": "products_777x4097x50_f32", "op": "products", "n": 777, "k": 4097, "dim": 50, "dtype": "float32"},
        # similarities of wide rows, the product itself in command
        {"name": "products_16384x8192x1024_bf16", "op": "products", "n": 16384, "k": 8192, "dim": 1024, "dtype": "bfloat16"},
        # how well the 512 picks of the small configuration cover it
        {"name": "coverage_20000x512x64", "op": "coverage", "n": 20000, "k": 512, "dim": 64, "prior": False},
        # a handful of new rows against a large selection: are they covered already? latency
        {"name": "coverage_33x16384x128", "op": "coverage", "n": 33, "k": 16384, "dim": 128, "prior": False},
        # a part of the single-GPU configuration's rows (256 wide) against its 10 000 picks
        {"name": "coverage_500000x10000x256", "op": "coverage", "n": 500000, "k": 10000, "dim": 256, "prior": True},
    ]


def _log(rng, low, high):
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["write", "read", "products", "coverage"])
    dim = _log(rng, 1, 1024)
    if rng.random() < 0.5:
        dim = min(1024, -(-dim // 16) * 16)
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    if op == "write":
        n = _log(rng, 1, min(2000000, 512000000 // dim))
        start = _log(rng, 1, 30000) - 1
        return {"op": op, "n": n, "dim": dim, "dtype": dtype, "capacity": start + n + _log(rng, 1, 1000) - 1, "start": start}
    if op == "read":
        n = _log(rng, 1, min(2000000, 1024000000 // dim))
        return {"op": op, "m": 0 if rng.random() < 0.4 else _log(rng, 1, n), "n": n, "dim": dim, "dtype": dtype}
    if op == "products":
        n = _log(rng, 1, 16384)
        k = _log(rng, 1, min(1000000, 134217728 // n))
        n, k = (n, k) if rng.random() < 0.5 else (k, n)
        return {"op": op, "n": n, "k": k, "dim": dim, "dtype": dtype}
    k = _log(rng, 1, 16384)
    n = _log(rng, 1, min(2000000, 1000000000 // k))
    return {"op": op, "n": n, "k": k, "dim": dim, "prior": rng.random() < 0.5}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _means(dim, g):
    return torch.randn(64, dim, generator=g, device="cuda") * 4


def _mixture(n, dim, g, means=None):
    """Rows of a mixture of 64 Gaussians, the shape of embeddings that clusters give: means N(0, 16), deviation 1."""
    means = _means(dim, g) if means is None else means
    x = torch.randn(n, dim, generator=g, device="cuda")
    return x.add_(means[torch.randint(0, 64, (n,), generator=g, device="cuda")])


def _power(e):
    """2^e of whole e in float32's normal range, exactly."""
    return ((e + BIAS) << 23).view(torch.float32)


def _quantise(x):
    """(codes, biased exponents, values) of float32 rows, by the definition."""
    n, dim = x.shape
    blocks = -(-dim // BLOCK)
    y = torch.nn.functional.pad(x, (0, blocks * BLOCK - dim)).view(n, blocks, BLOCK)
    fine = torch.isfinite(y)
    top, power = torch.frexp(torch.where(fine, y.abs(), 0.0).amax(2))
    e = torch.where(top <= 0.875, power - 9, power - 8)      # the least e with amax <= 448 * 2^e
    e = torch.where(top == 0, LOW, e).clamp_min(LOW).to(torch.int32)
    y = torch.where(fine, y, float("nan")) * _power(-e)[:, :, None]
    step = _power(torch.frexp(y)[1].to(torch.int32).clamp_min(-5) - 4)      # 3 bits behind the leading one, 2^-9 at least
    q = torch.round(y / step) * step
    value = (q * _power(e)[:, :, None]).view(n, -1)[:, :dim]
    return q.view(n, -1)[:, :dim].to(torch.float8_e4m3fn), (e + BIAS).to(torch.uint8), value


def _places(rows, dim, device):
    """Index arrays that say where the exponents of whole `rows` stand in `scales`."""
    blocks = torch.arange(-(-dim // BLOCK), device=device)[None]
    r = rows[:, None]
    return r // 128, blocks // 4, r % 32, r % 128 // 32, blocks % 4


def _empty_store(capacity, dim):
    pitch, words = -(-dim // 16) * 16, -(-dim // 512)
    return {
        "codes": torch.zeros(capacity, pitch, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
        "scales": torch.zeros(-(-capacity // 128), words, 32, 4, 4, dtype=torch.uint8, device="cuda"),
        "norms": torch.zeros(capacity, dtype=torch.float32, device="cuda"),
        "dim": dim,
    }


def _put(store, x, start):
    codes, exponents, value = _quantise(x.float())
    n, dim = x.shape
    store["codes"][start : start + n, :dim] = codes
    store["scales"][_places(torch.arange(start, start + n, device=x.device), dim, x.device)] = exponents
    store["norms"][start : start + n] = (value * value).sum(1)


def _filled(n, dim, g, means=None):
    means = _means(dim, g) if means is None else means
    store, rows = _empty_store(n, dim), 131072
    for a in range(0, n, rows):
        _put(store, _mixture(min(rows, n - a), dim, g, means), a)
    if own:
        from coresets_b200 import RowStore

        store["store"] = RowStore.from_tensors(store["codes"], store["scales"], store["norms"], dim)
    return store


def prepare(case, seed):
    g, op = _generator(seed), case["op"]
    s = {**case, "type": getattr(torch, case.get("dtype", "float32"))}
    if op == "write":
        s["into"] = _empty_store(case["capacity"], case["dim"])
        if own:
            from coresets_b200 import RowStore

            into = s["into"]
            into["store"] = RowStore.from_tensors(into["codes"], into["scales"], into["norms"], case["dim"])
        s["X"] = _mixture(case["n"], case["dim"], g).to(s["type"])
    elif op == "read":
        s["a"] = _filled(case["n"], case["dim"], g)
        s["rows"] = torch.randint(0, case["n"], (case["m"],), generator=g, device="cuda") if case["m"] else None
    else:
        means = _means(case["dim"], g)
        s["a"], s["b"] = (_filled(case[x], case["dim"], g, means) for x in "nk")
        if case.get("prior"):
            # what an earlier set of centres left: some rows nearer already, some selected (-1)
            h = torch.rand(case["n"], generator=g, device="cuda") * (4 * case["dim"])
            s["h"] = torch.where(torch.rand(case["n"], generator=g, device="cuda") < 0.01, -1.0, h)
    return s


def _values(store, rows=None):
    """The float32 rows that a store stands for."""
    codes, scales, dim = store["codes"], store["scales"], store["dim"]
    if rows is None:
        rows = torch.arange(codes.shape[0], device=codes.device)
        x = codes[:, :dim].float()
    else:
        x = codes.view(torch.uint8)[rows].view(torch.float8_e4m3fn)[:, :dim].float()
    power = _power(scales[_places(rows, dim, codes.device)].to(torch.int32) - BIAS)
    return x * power.repeat_interleave(BLOCK, 1)[:, :dim]


def run(s):
    op = s["op"]
    if own:
        import coresets_b200 as coresets

        if op == "write":
            coresets.quantise_rows(s["X"], store=s["into"]["store"], start=s["start"])
        elif op == "read":
            return coresets.read_rows(s["a"]["store"], s["rows"], dtype=s["type"])
        elif op == "products":
            return coresets.row_products(s["a"]["store"], s["b"]["store"], dtype=s["type"])
        else:
            return coresets.coverage(s["a"]["store"], s["b"]["store"], h=s.get("h"))
    elif op == "write":
        _put(s["into"], s["X"], s["start"])
    elif op == "read":
        return _values(s["a"], s["rows"]).to(s["type"])
    elif op == "products":
        return (_values(s["a"]) @ _values(s["b"]).T).to(s["type"])
    else:
        a, b = s["a"], s["b"]
        d = _values(a) @ _values(b).T
        d = d.mul_(-2).add_(a["norms"][:, None]).add_(b["norms"]).amin(1).clamp_min(0)
        return d if "h" not in s else torch.minimum(s["h"], d, out=s["h"])
    into, first, last = s["into"], s["start"], s["start"] + s["n"]
    return {
        "codes": into["codes"][first:last, : s["dim"]],
        "scales": into["scales"][first // 128 : (last - 1) // 128 + 1],
        "norms": into["norms"][first:last],
    }


def work(case):
    op, dim = case["op"], case["dim"]
    row = dim + -(-dim // BLOCK)          # a stored row without its norm
    if op == "write":
        return {"bytes": case["n"] * (dim * SIZES[case["dtype"]] + row + 4), "flops": 0}
    if op == "read":
        m = case["m"] or case["n"]
        return {"bytes": m * (row + dim * SIZES[case["dtype"]] + (8 if case["m"] else 0)), "flops": 0}
    n, k = case["n"], case["k"]
    if op == "products":
        return {"bytes": (n + k) * row + n * k * SIZES[case["dtype"]], "flops": 2 * n * k * dim}
    return {"bytes": (n + k) * (row + 4) + n * (8 if case["prior"] else 4), "flops": 2 * n * k * dim}


def _code_values():
    """The 256 numbers that an e4m3 byte stands for, from its bits: sign, 4 bits of exponent (bias 7), 3 of fraction."""
    table = []
    for c in range(256):
        power, part = c >> 3 & 15, c & 7
        v = part / 512 if power == 0 else (1 + part / 8) * 2.0 ** (power - 7)
        table.append((float("nan") if c & 127 == 127 else v) * (-1 if c >> 7 else 1))
    return torch.tensor(table, dtype=torch.float64, device="cuda")


def _exact_power(e):
    """2^e of whole e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_rows(store, rows):
    """The rows that a store stands for, in 64 bits."""
    value = _code_values()[store["codes"].view(torch.uint8)[rows].long()][:, : store["dim"]]
    flat = store["scales"].permute(0, 3, 2, 1, 4).flatten(0, 2).flatten(1)[rows].double()
    place = torch.arange(store["dim"], device="cuda") // BLOCK
    return value * _exact_power(flat[:, place] - BIAS)


def exact(case, seed):
    s, op, dim = prepare(case, seed), case["op"], case["dim"]
    if op == "write":
        x, n = s["X"].double(), case["n"]
        first, last = case["start"], case["start"] + n
        mags = _code_values()[:127]                        # 0 .. 448, rising
        codes = torch.empty(n, dim, dtype=torch.float64, device="cuda")
        exps = torch.empty(n, -(-dim // BLOCK), dtype=torch.int64, device="cuda")
        norms = torch.zeros(n, dtype=torch.float64, device="cuda")
        for b in range(exps.shape[1]):
            for a in range(0, n, 262144):
                part = x[a : a + 262144, b * BLOCK : (b + 1) * BLOCK]
                top = part.abs().amax(1)
                e = torch.ceil(torch.log2(top / 448).nan_to_num(neginf=LOW)).clamp_min(LOW)
                e = torch.where(top > 448 * _exact_power(e), e + 1, e)          # whatever log2 rounded
                e = torch.where((e > LOW) & (top <= 448 * _exact_power(e - 1)), e - 1, e)
                scaled = part.abs() / _exact_power(e)[:, None]
                up = torch.bucketize(scaled, mags).clamp(1, 126)
                low, high = scaled - mags[up - 1], mags[up] - scaled
                near = torch.where((high < low) | ((high == low) & (up % 2 == 0)), up, up - 1)   # a tie goes to the even code
                q = mags[near] * part.sign()
                codes[a : a + 262144, b * BLOCK : (b + 1) * BLOCK] = q
                exps[a : a + 262144, b] = e.long() + BIAS
                norms[a : a + 262144] += (q * _exact_power(e)[:, None]).square().sum(1)
        scales = s["into"]["scales"]
        rows = torch.arange(first, last, device="cuda")
        for b in range(exps.shape[1]):
            scales[rows // 128, b // 4, rows % 32, rows % 128 // 32, b % 4] = exps[:, b].to(torch.uint8)
        return {"codes": codes, "scales": scales[first // 128 : (last - 1) // 128 + 1], "norms": norms}
    if op == "read":
        rows = torch.arange(case["n"], device="cuda") if s["rows"] is None else s["rows"]
        return torch.cat([_exact_rows(s["a"], rows[a : a + 65536]) for a in range(0, len(rows), 65536)])
    a_rows, b = torch.arange(case["n"], device="cuda"), _exact_rows(s["b"], torch.arange(case["k"], device="cuda"))
    if op == "products":
        return torch.cat([_exact_rows(s["a"], r) @ b.T for r in a_rows.split(16384)])
    # |a|^2 + |b|^2 - 2 a.b in 64 bits: the cancellation leaves 1e-13 of the norms
    b_norms, out = b.square().sum(1), []
    for r in a_rows.split(max(1, 1 << 28) // case["k"] + 1):
        a = _exact_rows(s["a"], r)
        out.append((a.square().sum(1) + (b_norms - 2 * (a @ b.T)).amin(1)).clamp_min(0))
    d = torch.cat(out)
    return torch.minimum(s["h"].double(), d) if "h" in s else d
