"""Pages that several sequences hold: what the documents promise of them, and the pattern that they name, with a plain loop in the place of the kernels."""
import os
import re

from tests.test_gpu_pages import plain_cut, plain_take

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_documents_exclude_cuts_of_shared_pages():
    """Nobody counts a page's users: whoever reads of shared pages reads that too."""
    import amdgpu_rustdsl_b200 as A
    words = lambda text: re.sub(r"[\s*]+", " ", text)
    read = lambda *at: words(open(os.path.join(ROOT, *at)).read())
    for text in (read("include", "fmha_pages_abi.h"), words(A.pages_cut.__doc__)):
        assert "Nobody counts a page's users" in text and "in front of" in text
    assert "does not count their users" in words(A.kv8_append.__doc__) and "counts no users" in read("INTEGRATION.md")


def test_a_prefix_in_common_stays_where_it_is():
    """Two sequences share a full page; one ends with keep at the prefix's end: a third is handed other pages."""
    page, free, table, lengths = 16, [3, 0, 0, 0, 4, 3, 2, 0], [[0, 1, -1], [0, -1, -1], [-1, -1, -1]], [30, 16, 0]
    plain_cut(free, table, lengths, [16, 16, 0], page)
    assert table == [[0, -1, -1], [0, -1, -1], [-1, -1, -1]] and free[0] == 4
    plain_take(free, table, lengths, [0, 0, 48], page, 1)
    assert 0 not in table[2] and sorted(table[2]) == [1, 2, 3]


def test_what_a_cut_behind_it_would_do():
    """The same with keep of 0: the shared page goes to the third, while the second sequence still reads it. This is what the documents exclude."""
    page, free, table, lengths = 16, [0, 0, 0, 0, 9, 9], [[0], [0], [-1]], [16, 16, 0]
    plain_cut(free, table, lengths, [0, 16, 0], page)
    plain_take(free, table, lengths, [0, 0, 16], page, 1)
    assert table == [[-1], [0], [0]]
