"""The GPT app's generation over a paged cache (gpt paged-check, beam-check, generate --beams / --budget;
PagedKVCache and beam_select of the C++ layer) on the GPU.

A cache that never fills: the logits at every position against the oracle's causal forward of the whole
sequence (oracle/gpt.py, the reference chain per layer).  A bounded one: against a plain simulation in 64
bits that keeps, per layer and head, the same positions.  Beam search: every step's picks against the
oracle's logits of the sequences that the beams stand for.

Bar: max|x - ref| / max|ref| <= 1e-4 per position, as for the contiguous cache; a beam's score sums
N log-probabilities, each off by twice a logit's error at most.
"""
import math
import subprocess
from pathlib import Path

import numpy as np
import pytest

from oracle import gpt as ogpt

ROOT = Path(__file__).resolve().parents[1]
APP = ROOT / "inferno_amd" / "gpt"
TOL = 1e-4


def write_case(tmp_path, L, C, H, T, V, B, seed=5):
    params = ogpt.init_params(L, C, V, seed=seed)
    (tmp_path / "config.txt").write_text(f"{L} {C} {H} {T} {V} {B}\n")
    for name, val in params.items():
        np.ascontiguousarray(val, np.float32).tofile(tmp_path / f"{name}.bin")
    return params


def run_app(*args, ok=True):
    if not APP.exists():
        pytest.skip("inferno_amd/gpt not built")
    r = subprocess.run([str(APP), *map(str, args)], capture_output=True, text=True, timeout=600)
    assert (r.returncode == 0) == ok, r.stdout + r.stderr
    return r.stdout + r.stderr


def tokens_file(tmp_path, V, B, n, seed=11):
    tokens = np.random.default_rng(seed).integers(0, V, size=(B, n), dtype=np.int32)
    tokens.tofile(tmp_path / "tokens.bin")
    return tokens


def test_cpu_is_refused(tmp_path):
    """The paged cache lives on a HIP device: the CPU is refused with a message, before any work."""
    write_case(tmp_path, 1, 32, 1, 12, 20, 2)
    tokens_file(tmp_path, 20, 2, 12)
    for cmd in ("paged-check", "beam-check"):
        assert "HIP device" in run_app(cmd, tmp_path, "cpu", ok=False)


@pytest.mark.gpu
@pytest.mark.parametrize("P,page", [(1, 16), (7, 4), (33, 64), (70, 1)])
def test_paged_cache_never_full(tmp_path, P, page):
    print(f"[case] paged cache prompt {P} page {page}", flush=True)
    L, C, H, T, V, B = 2, 128, 2, 70, 96, 3
    params = write_case(tmp_path, L, C, H, T, V, B)
    tokens = tokens_file(tmp_path, V, B, T)
    run_app("paged-check", tmp_path, "hip", "--prompt", P, "--page-size", page)
    got = np.fromfile(tmp_path / "paged_logits.bin", np.float32).reshape(B, T - P + 1, V)
    ref = ogpt.gpt_logits(params, tokens, L, C, H)[:, P - 1:]
    assert np.abs(got.astype(np.float64) - ref).max() <= TOL * np.abs(ref).max()


def layer_norm(x, g, b):
    m = x.mean(-1, keepdims=True)
    return (x - m) / np.sqrt(((x - m) ** 2).mean(-1, keepdims=True) + 1e-5) * g + b


def simulate(params, tokens, L, C, H, P, capacity, keep, recent):
    """Logits from the prompt's last position on, one sequence, in 64 bits, with the bounded cache's rule."""
    p = {k: v.astype(np.float64) for k, v in params.items()}
    D, T = C // H, tokens.shape[0]
    pe = ogpt.positional_encoding(T, C).astype(np.float64)
    held = [[[] for _ in range(H)] for _ in range(L)]  # [position, k, v, weight] by slot
    out = []
    for pos in range(T):
        if pos >= P and len(held[0][0]) == capacity:
            for layer in held:
                for h in range(H):
                    mine = layer[h]
                    newest = max(m[0] for m in mine)
                    rank = sorted(range(len(mine)),
                                  key=lambda j: (0, 0.0, j) if mine[j][0] > newest - recent else (1, -mine[j][3], j))
                    kept = set(rank[:keep])
                    holes = [j for j in range(keep) if j not in kept]
                    for a, b in zip(holes, [j for j in range(keep, len(mine)) if j in kept]):
                        mine[a] = mine[b]
                    del mine[keep:]
        x = p["tok_embedding.weight"][tokens[pos]] + pe[pos]
        for i in range(L):
            q = lambda s: p[f"block{i}.{s}"]  # noqa: B023,E731
            n = layer_norm(x, q("ln1.gamma"), q("ln1.beta"))
            qkv = n @ q("attn.Wqkv.weights") + q("attn.Wqkv.bias")
            o = np.zeros(C)
            for h in range(H):
                s = slice(h * D, (h + 1) * D)
                mine = held[i][h]
                mine.append([pos, qkv[C:2 * C][s], qkv[2 * C:][s], 0.0])
                e = np.array([m[1] for m in mine]) @ qkv[:C][s] / math.sqrt(D)
                e = np.exp(e - e.max())
                e /= e.sum()
                o[s] = e @ np.array([m[2] for m in mine])
                if pos >= P or P == 1:  # the prompt's attention runs without the cache
                    for m, w in zip(mine, e):
                        m[3] += w
            x = x + o @ q("attn.W_out.weights") + q("attn.W_out.bias")
            n = layer_norm(x, q("ln2.gamma"), q("ln2.beta"))
            a = n @ q("ff1.weights") + q("ff1.bias")
            a = 0.5 * a * (1 + np.tanh(0.7978845608028654 * (a + 0.044715 * a**3)))
            x = x + a @ q("ff2.weights") + q("ff2.bias")
        if pos >= P - 1:
            out.append(layer_norm(x, p["ln1.gamma"], p["ln1.beta"]) @ p["tok_embedding.weight"].T)
    return np.array(out)


@pytest.mark.gpu
@pytest.mark.parametrize("P,capacity,keep,recent,page", [(9, 24, 16, 4, 8), (1, 20, 19, 3, 1), (30, 32, 8, 8, 16)])
def test_paged_cache_bounded(tmp_path, P, capacity, keep, recent, page):
    print(f"[case] paged cache cut from {capacity} to {keep}", flush=True)
    L, C, H, T, V, B = 2, 128, 2, 90, 96, 2
    params = write_case(tmp_path, L, C, H, T, V, B, seed=7)
    tokens = tokens_file(tmp_path, V, B, T)
    run_app("paged-check", tmp_path, "hip", "--prompt", P, "--capacity", capacity, "--budget", keep, "--recent", recent,
            "--page-size", page)
    got = np.fromfile(tmp_path / "paged_logits.bin", np.float32).reshape(B, T - P + 1, V)
    for b in range(B):
        ref = simulate(params, tokens[b], L, C, H, P, capacity, keep, recent)
        assert np.abs(got[b].astype(np.float64) - ref).max() <= TOL * np.abs(ref).max()


@pytest.mark.gpu
def test_paged_cache_refusals(tmp_path):
    print("[case] paged cache refusals", flush=True)
    write_case(tmp_path, 1, 64, 1, 40, 30, 2)
    tokens_file(tmp_path, 30, 2, 40)
    assert "full" in run_app("paged-check", tmp_path, "hip", "--capacity", 20, ok=False)
    assert "longer" in run_app("paged-check", tmp_path, "hip", "--capacity", 20, "--prompt", 30, ok=False)
    assert "budget" in run_app("paged-check", tmp_path, "hip", "--capacity", 20, "--budget", 20, ok=False)
    assert "recent" in run_app("paged-check", tmp_path, "hip", "--capacity", 20, "--budget", 8, "--recent", 9, ok=False)
    assert "power of two" in run_app("paged-check", tmp_path, "hip", "--page-size", 12, ok=False)
    assert "32 beams" in run_app("beam-check", tmp_path, "hip", "--beams", 33, ok=False)


@pytest.mark.gpu
@pytest.mark.parametrize("P,K,page,eos", [(5, 4, 4, -1), (1, 3, 16, -1), (8, 5, 8, 3), (6, 1, 2, -1)])
def test_beam_search(tmp_path, P, K, page, eos):
    print(f"[case] beam search prompt {P} beams {K} page {page} eos {eos}", flush=True)
    L, C, H, T, V, B, N = 2, 64, 2, 40, 50, 2, 20
    params = write_case(tmp_path, L, C, H, T, V, B, seed=21)
    prompt = tokens_file(tmp_path, V, B, P, seed=12)
    args = ["--prompt", P, "--new", N, "--beams", K, "--page-size", page] + (["--eos", eos] if eos >= 0 else [])
    run_app("beam-check", tmp_path, "hip", *args)
    tok, par = (np.fromfile(tmp_path / f"beam_{n}.bin", np.int32).reshape(N, B, K) for n in ("tokens", "parents"))
    scores = np.fromfile(tmp_path / "beam_scores.bin", np.float32).reshape(N, B, K).astype(np.float64)
    seqs = [[list(prompt[b]) for _ in range(K)] for b in range(B)]
    done = np.zeros((B, K), bool)
    before = np.full((B, K), -np.inf)
    before[:, 0] = 0.0
    for step in range(N):
        for b in range(B):
            logits = ogpt.gpt_logits(params, np.array(seqs[b], np.int32), L, C, H)[:, -1].astype(np.float64)
            err = 2 * TOL * np.abs(logits).max()  # of a log-probability
            lp = logits - logits.max(1, keepdims=True)
            lp -= np.log(np.exp(lp).sum(1, keepdims=True))
            lp[done[b]] = -np.inf
            if eos >= 0:
                lp[done[b], eos] = 0.0
            every = before[b][:, None] + lp
            best = np.sort(every.ravel())[::-1][:K]
            mine = every[par[step, b], tok[step, b]]
            assert np.isfinite(mine).all()
            assert np.abs(mine - best).max() <= 2 * err and np.abs(scores[step, b] - mine).max() <= err + 1e-5
            assert len({(p, t) for p, t in zip(par[step, b], tok[step, b])}) == K
            seqs[b] = [seqs[b][p] + [int(t)] for p, t in zip(par[step, b], tok[step, b])]
            done[b] = [done[b][p] or t == eos for p, t in zip(par[step, b], tok[step, b])]
        before = scores[step]
    final = np.fromfile(tmp_path / "beams.bin", np.int32).reshape(B, K, N)
    assert (final == np.array([[s[P:] for s in seqs[b]] for b in range(B)])).all()


@pytest.mark.gpu
def test_generate_commands():
    print("[case] generate over a paged cache", flush=True)
    small = ["--layers", 2, "--dmodel", 128, "--heads", 2, "--vocab", 128, "--batch", 2, "--prompt", 20, "--new", 30,
             "--ctx", 64]
    plain, bounded = run_app("generate", *small), run_app("generate", *small, "--budget", 63, "--capacity", 64)
    first = [line.split("first_tokens")[1] for line in (plain, bounded)]
    assert first[0] == first[1]  # nothing was cut
    assert "cut to 16" in run_app("generate", *small, "--budget", 16)
    assert "best_score" in run_app("generate", *small, "--beams", 3, "--page-size", 8)
    assert "exclude" in run_app("generate", *small, "--beams", 3, "--budget", 16, ok=False)
