"""PagedKVCache of the C++ layer on given queries, keys and values, in both types, against a plain simulation in 64
bits: prompts, steps, beams that are reordered, and a bounded cache.

Tolerance of a step's output: with A = max sum |q_d k_d| scale of a row, a score is off by (D + 2) 2^-24 A and its
exponent's argument by two roundings more, so a probability by 2 ((D + 2) + 4.5) 2^-24 A + 2^-22 of itself and sums over n
by (n / 16 + 64) 2^-24; bf16 probabilities in two parts add 2^-16, bf16 outputs 2^-8 of themselves.  The prompt goes
through the contiguous attention, whose bar is 1e-4 (fp32) and 2e-2 (bf16) of the largest output.  A bounded cache
evicts by sums of probabilities, which the cases' seeds keep further apart than their error (asserted).
"""
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

DRIVER = Path(__file__).resolve().parent / "cpp" / "paged_driver"


def rel_err(a, D, n, bf16):
    return 2 * (D + 6.5) * 2.0**-24 * a + 2.0**-22 + (n / 16 + 64) * 2.0**-24 + (2.0**-16 if bf16 else 0.0)


CASES = [
    # groups, beams, H, D, prompt, steps, page, capacity, budget, recent
    (3, 1, 2, 64, 7, 12, 4, 32, 0, 0),
    (2, 1, 3, 128, 1, 40, 16, 48, 0, 0),
    (2, 4, 2, 32, 21, 30, 8, 64, 0, 0),
    (1, 3, 1, 128, 16, 20, 16, 40, 0, 0),
    (2, 1, 2, 64, 20, 40, 8, 24, 14, 4),
    (1, 1, 3, 128, 9, 60, 1, 20, 19, 0),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("G,K,H,D,P,S,page,capacity,budget,recent", CASES)
def test_cache(tmp_path, G, K, H, D, P, S, page, capacity, budget, recent, dtype):
    if not DRIVER.exists():
        pytest.skip("paged_driver not built")
    print(f"[case] PagedKVCache {G}x{K} H{H} D{D} prompt {P} steps {S} budget {budget} {dtype}", flush=True)
    L, R, bf16, scale = 2, G * K, dtype == "bf16", D**-0.5
    gen = torch.Generator().manual_seed(1000 * D + P)
    x = {n: torch.randn(L, G, H, P, D, generator=gen) for n in ("q", "k", "v")}
    x |= {n: torch.randn(S, L, R, H, 1, D, generator=gen) for n in ("sq", "sk", "sv")}
    x["q"], x["sq"] = x["q"] * 1.5, x["sq"] * 1.5
    for n in x:
        if bf16:
            x[n] = x[n].bfloat16().float()
        x[n].numpy().tofile(tmp_path / f"{n}.bin")
        x[n] = x[n].double().numpy()
    parents = torch.randint(0, K, (S, G, K), generator=gen, dtype=torch.int32).numpy()
    parents.tofile(tmp_path / "parents.bin")
    r = subprocess.run([str(DRIVER), str(tmp_path), dtype, *map(str, (G, K, L, H, D, P, S, page, capacity, budget, recent))],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    o = np.fromfile(tmp_path / "o.bin", np.float32).reshape(L, G, H, P, D).astype(np.float64)
    so = np.fromfile(tmp_path / "so.bin", np.float32).reshape(S, L, R, H, D).astype(np.float64)

    # the prompt
    s = x["q"] @ x["k"].swapaxes(-1, -2) * scale
    s[..., np.triu(np.ones((P, P), bool), 1)] = -np.inf
    p = np.exp(s - s.max(-1, keepdims=True))
    want = p / p.sum(-1, keepdims=True) @ x["v"]
    assert np.abs(o - want).max() <= (2e-2 if bf16 else 1e-4) * np.abs(want).max()

    # [position, key, value, weight, the weight's error] by slot
    start = 1.0 if P == 1 else 0.0  # a prompt of one token is a step
    held = [[[[[j, x["k"][l, g, h, j], x["v"][l, g, h, j], start, start * 2.0**-20] for j in range(P)] for h in range(H)]
             for g in range(G) for _ in range(K)] for l in range(L)]
    seen, cuts = P, 0
    for step in range(S):
        if K > 1:
            pick = [g * K + int(b) for g in range(G) for b in parents[step, g]]
            held = [[[[m[:] for m in held[l][i][h]] for h in range(H)] for i in pick] for l in range(L)]
        cut = len(held[0][0][0]) == capacity
        cuts += cut
        for l in range(L):
            for row in range(R):
                for h in range(H):
                    mine = held[l][row][h]
                    if cut:
                        newest = max(m[0] for m in mine)
                        safe = [m[0] > newest - recent for m in mine]
                        rank = sorted(range(len(mine)), key=lambda j: (0, 0.0, j) if safe[j] else (1, -mine[j][3], j))
                        kept, gone = rank[:budget], rank[budget:]
                        if not safe[kept[-1]]:  # the last one kept and the first one gone: apart, or equal for sure
                            a, b = mine[kept[-1]], mine[gone[0]]
                            assert a[3] - b[3] > a[4] + b[4] or a[3] == b[3] == 0.0
                        holes = [j for j in range(budget) if j not in kept]
                        for a, b in zip(holes, [j for j in range(budget, len(mine)) if j in kept]):
                            mine[a] = mine[b]
                        del mine[budget:]
                    mine.append([seen, x["sk"][step, l, row, h, 0], x["sv"][step, l, row, h, 0], 0.0, 0.0])
                    q = x["sq"][step, l, row, h, 0]
                    kk, vv = np.array([m[1] for m in mine]), np.array([m[2] for m in mine])
                    e = kk @ q * scale
                    w = np.exp(e - e.max())
                    w /= w.sum()
                    rel = rel_err(float((np.abs(kk) @ np.abs(q)).max() * scale), D, len(mine), bf16)
                    want = w @ vv
                    bound = rel * (w @ np.abs(vv)).max() + (2.0**-8 * np.abs(want) if bf16 else 0.0)
                    assert (np.abs(so[step, l, row, h] - want) <= bound).all(), (step, l, row, h)
                    for m, v in zip(mine, w):
                        m[3] += v
                        m[4] += rel * v + 2.0**-24 * m[3]
        seen += 1
    assert f"length {len(held[0][0][0])} seen {P + S}" in r.stdout
    assert not budget or cuts > 1
    assert math.isfinite(float(so.sum()))
