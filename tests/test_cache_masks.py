"""The mask functions of pa_cache.cuh compiled as host code: for random windows, sinks, lengths, positions and trees,
vis64 of every 64-key group says, bit for bit, what the definition says, and the groups of span_of hold every visible key
once. Also the refusals that need no GPU."""
import os
import random
import subprocess

import pytest

import backburner_b200 as pa

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SRC = r'''
#include <cstdio>
#include <cstdlib>
#include "pa_mask.cuh"
using namespace pa::pg;
template <int G> void spans(const View &v, Set st, unsigned t0, unsigned t1) {
  Span p = span_of<G>(v, st, t0, t1);
  printf("G %d", p.n);
  for (int i = 0; i < p.n; i++) printf(" %d", p.group(i));
  printf("\n");
}
int main() {
  int n_tok, window, sinks, tree, n, q0, cap;
  while (scanf("%d %d %d %d %d %d %d", &n_tok, &window, &sinks, &tree, &n, &q0, &cap) == 7) {
    uint64_t bits[64];
    for (int t = 0; t < n_tok && tree; t++) { unsigned long long x; if (scanf("%llu", &x) != 1) return 1; bits[t] = x; }
    View v{};
    v.tree = tree ? bits : nullptr; v.n_sets = 1; v.max_pages = cap / 64; v.page_keys = 64; v.n_tok = n_tok;
    v.window = window; v.sinks = sinks;
    Set st{clampi(n, 0, capacity(v)), q0};
    for (int t = 0; t < n_tok; t++) {
      Row r = row_of(v, st, 0, t);
      printf("R");
      for (int k0 = 0; k0 < cap; k0 += 64) printf(" %llx", (unsigned long long) vis64(r, k0));
      printf("\n");
    }
    spans<64>(v, st, 0, n_tok - 1);
    spans<16>(v, st, 0, n_tok - 1);
    spans<64>(v, st, n_tok / 2, n_tok / 2);
  }
  return 0;
}
'''


def _sees(n_tok, window, sinks, bits, n, q0, t, j):
    if j < 0 or j >= n:
        return False
    if bits is None:
        at = q0 + t
        return j <= at and (not window or j > at - window or j < sinks)
    b = bits[t] & ((1 << n_tok) - 1)
    if not b:
        return False
    if j < q0:
        at = q0 + bin(b).count("1") - 1
        return not window or j > at - window or j < sinks
    return j - q0 < n_tok and bool(b >> (j - q0) & 1)


def test_masks_are_the_definition(tmp_path):
    src, exe = tmp_path / "m.cu", tmp_path / "m"
    src.write_text(SRC)
    nvcc = "/usr/local/cuda/bin/nvcc" if os.path.exists("/usr/local/cuda/bin/nvcc") else "nvcc"
    r = subprocess.run([nvcc, "-std=c++17", "-I", os.path.join(ROOT, "backburner_b200", "csrc"), "-o", str(exe), str(src)],
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    rng, cases, text = random.Random(7), [], []
    for i in range(400):
        tree = rng.random() < 0.5
        n_tok = rng.choice([1, 2, 7, 63, 64]) if tree else rng.choice([1, 2, 9, 70])
        n = rng.choice([0, 1, 5, 63, 64, 65, 128, 200, 300, 320])
        window = rng.choice([0, max(1, n_tok if tree else 1), 64, 65, 100, 1 << 30])
        if tree and window and window < n_tok:
            window = n_tok
        sinks = 0 if not window else rng.choice([0, 1, 4, 64, 65, 130, 1 << 30, (1 << 32) - 1])
        q0 = rng.choice([n - n_tok, n - n_tok, n, n + 50, 0, -3, -100, 2**31 - 1, -2**31, n - 1])
        bits = None
        if tree:
            bits = []
            for t in range(n_tok):
                p = rng.randrange(-1, t)
                bits.append(0 if rng.random() < 0.2 else (1 << t) | (bits[p] if p >= 0 else 0))
        cases.append((n_tok, window, sinks, bits, n, q0))
        text.append(" ".join(map(str, (n_tok, window, sinks if sinks < 2**31 else -1, int(tree), n, q0, 320))) +
                    "".join(f" {b}" for b in bits or []))
    out = subprocess.run([str(exe)], input="\n".join(text), capture_output=True, text=True)
    assert out.returncode == 0
    lines = iter(out.stdout.splitlines())
    for n_tok, window, sinks, bits, n, q0 in cases:
        seen = set()
        per_tok = []
        for t in range(n_tok):
            words = [int(x, 16) for x in next(lines).split()[1:]]
            got = {64 * g + b for g, w in enumerate(words) for b in range(64) if w >> b & 1}
            want = {j for j in range(320) if _sees(n_tok, window, sinks, bits, n, q0, t, j)}
            assert got == want, (n_tok, window, sinks, bits, n, q0, t)
            per_tok.append(want)
            seen |= want
        for G, keys in ((64, seen), (16, seen), (64, per_tok[n_tok // 2])):
            groups = [int(x) for x in next(lines).split()[2:]]
            assert len(set(groups)) == len(groups) and groups == sorted(groups)
            assert keys <= {G * g + i for g in groups for i in range(G)}, (G, n_tok, window, sinks, bits, n, q0)
            assert all(0 <= G * g < max(n, 1) for g in groups)


class _Ctx:
    device, handle = 0, None


def test_refusals_without_a_gpu():
    import torch
    cpu = torch.zeros((1, 1, 64, 1088), dtype=torch.uint8)
    for K, V in ((cpu, cpu), (cpu.float(), cpu), (cpu[0], cpu[0])):
        with pytest.raises(pa.PaCudaError):
            pa.Cache.of(K, V, hd=128, nkv=8, quant=pa.Q8_0)
    from backburner_b200 import api
    for t, dtype, shape in ((torch.zeros(3, dtype=torch.int32), torch.int32, (3,)),          # on the CPU
                            (torch.zeros(3, dtype=torch.int64), torch.int32, (3,)),
                            (torch.zeros(4, dtype=torch.int32), torch.int32, (3,)),
                            (torch.zeros(6, dtype=torch.int32)[::2], torch.int32, (3,))):
        with pytest.raises(pa.PaCudaError) as e:
            api._want(_Ctx, t, "table", dtype, shape)
        assert e.value.code == api.EINVAL and "table" in str(e.value)
    L = pa.lib()
    assert L.pa_cuda_cache_plan_create(None, None, None, 1, 1, None, None) == api.EINVAL
    assert L.pa_cuda_cache_attn(None, 0, None, None, None, None, None, None, None, None, None) == api.EINVAL
    assert L.pa_cuda_cache_attn_reply(None, 0, None, None, None, None, None, None, None, None) == api.EINVAL
    assert L.pa_cuda_cache_append(None, None, None, 0, None, 1, 1, None, 1, None, None, None) == api.EINVAL
    assert L.pa_cuda_cache_rows(None, None, None, 0, 1, 1, None, 1, None, None, None, None) == api.EINVAL
    assert L.pa_cuda_cache_copy_pages(None, None, None, None, None, 1, None) == api.EINVAL
    assert L.pa_cuda_cache_compact(None, None, None, 1, 1, None, 1, None, None, None, None, None) == api.EINVAL
    L.pa_cuda_cache_plan_destroy(None)
