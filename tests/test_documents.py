"""The ranges of packed documents, on the CPU, row by row against what the words of ``documents`` say."""

import pytest
import torch

from cqgdn import attention


def said(bounds, causal, window, prefix):
    rows = []
    for i, (a, b) in enumerate(zip(bounds, bounds[1:])):
        for t in range(a, b):
            seen = [j for j in range(a, b) if (j <= t or not causal) and (window is None or abs(t - j) < window)]
            if prefix is not None and t < a + prefix[i]:
                seen += [j for j in range(t + 1, min(b, a + prefix[i])) if j not in seen]
            assert sorted(seen) == list(range(min(seen), max(seen) + 1))
            rows.append((min(seen), max(seen) + 1))
    return rows


@pytest.mark.parametrize("prefix", [None, (0, 3, 1, 0, 20)])
@pytest.mark.parametrize("window", [None, 1, 2, 5, 8, 100])
@pytest.mark.parametrize("causal", [False, True])
def test_documents_row_by_row(causal, window, prefix):
    bounds = [0, 1, 9, 9, 15, 26]
    first, limit = attention.documents(bounds, causal=causal, window=window, prefix=prefix, device="cpu")
    assert list(zip(first.tolist(), limit.tolist())) == said(bounds, causal, window, prefix)
    assert first.dtype == limit.dtype == torch.int32
