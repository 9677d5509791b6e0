"""CPU: the synthetic matrices are the same whether their chunks are worked on one after another or by several threads."""
import numpy as np
import pytest
import scipy.sparse as sp

from sclens_amd import synth


def parameters(rng, N, M, C, sparsity):
    beta0, delta = synth._rates(M, C, rng)
    lo, hi = -8.0, 8.0
    for _ in range(60):
        mid = 0.5 * (lo + hi)
        lo, hi = (mid, hi) if synth._sparsity_for_offset(beta0, mid) > sparsity else (lo, mid)
    labels = np.arange(N) % C
    rng.shuffle(labels)
    return beta0 + 0.5 * (lo + hi), delta, labels, rng.lognormal(0.0, 0.3, size=N)


def same(X, dense):
    ref = sp.csc_matrix(dense)
    ref.sort_indices()
    assert X.format == "csc" and X.dtype == np.float32 and X.indices.dtype == np.int32 and X.has_sorted_indices
    assert np.array_equal(X.indptr, ref.indptr) and np.array_equal(X.indices, ref.indices) and np.array_equal(X.data, ref.data)


@pytest.mark.parametrize("N,M,chunk", [(997, 301, 100), (64, 200, 64), (700, 90, 37), (300, 50, 4096)])
def test_counts_follow_one_generator(N, M, chunk):
    """nothing planted: the draws of one generator, chunk after chunk"""
    rng = np.random.Generator(np.random.PCG64(11))
    beta0, delta, labels, lib = parameters(rng, N, M, 4, 0.7)
    dense = np.concatenate([rng.poisson(lib[a:a + chunk, None] * np.exp(beta0[None, :] + delta[labels[a:a + chunk]])) for a in range(0, N, chunk)])
    same(synth.synth_counts(N, M, seed=11, C=4, sparsity=0.7, chunk_rows=chunk, min_genes_per_cell=0, min_cells_per_gene=0), dense.astype(np.float32))


@pytest.mark.parametrize("a,b", [(0, 1000), (130, 777), (256, 257), (999, 1000)])
def test_rows_have_a_generator_per_chunk(a, b):
    N, M, chunk, mg = 1000, 120, 64, 5
    beta0, delta, labels, lib = parameters(np.random.Generator(np.random.PCG64(3)), N, M, 8, 0.95)
    out = []
    for c in range(0, (N + chunk - 1) // chunk):
        r = slice(c * chunk, min(N, (c + 1) * chunk))
        rng = np.random.Generator(np.random.PCG64([3, c]))
        x = rng.poisson(lib[r, None] * np.exp(beta0[None, :] + delta[labels[r]])).astype(np.float32)
        for i in np.flatnonzero((x > 0).sum(axis=1) < mg):
            x[i, rng.choice(np.flatnonzero(x[i] == 0), size=mg - int((x[i] > 0).sum()), replace=False)] = 1.0
        out.append(x)
    same(synth.synth_counts_rows(N, M, 3, a, b, sparsity=0.95, chunk_rows=chunk, min_genes_per_cell=mg), np.concatenate(out)[a:b])
