"""Deep forks of rows with holes: what they need and what they leave free."""
import pytest

from moearc_b200 import Context
from paged_model import FULL, NO_PAGE
from test_gpu_kvcache import Pair

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = Context()
    yield c
    c.close()


@pytest.mark.parametrize("pages", [7, 8])
def test_a_deep_fork_needs_a_free_page_for_every_table_entry(ctx, pages):
    """Four entries, two of them holes: with four free pages the row is copied onto two of them and the ones
    passed over stay free; with three it cannot be done and nothing changes."""
    p = Pair(ctx, pages=pages, pt=4, rows=4, max_pages=6)
    p.do("grow", [1, 0, 2], [4, 14, 4])  # pages 0, 1 to 4 and 5
    for j in (0, 2):
        p.m.refs[p.m.tables[0][j]] -= 1
        p.m.tables[0][j] = NO_PAGE
    p.put()  # free: 1, 3, 6 (and 7)
    was = [list(r) for r in p.m.tables], list(p.m.refs)
    p.do("fork", [0], [3], deep=True)
    if pages == 7:
        assert p.m.status == FULL and (p.m.tables, p.m.refs) == was
    else:
        assert p.m.status == 0 and p.m.tables[3][:4] == [NO_PAGE, 3, NO_PAGE, 7]
        assert p.m.refs[1] == p.m.refs[6] == 0
    p.same()
    p.do("fork", [0], [3])  # shared, but for the last page; onto a row that is taken in the other case
    p.same()
