"""The book of a pool's blocks: allocation, shared users, forks, blocks behind a
window given back (host only)."""
import random

import pytest

import fmkv


def test_alloc_and_release():
    book = fmkv.PageBook(5)
    a = book.alloc(3)
    assert len(set(a)) == 3 and all(0 <= b < 5 for b in a) and book.free_count() == 2
    assert [book.users(b) for b in a] == [1, 1, 1]
    with pytest.raises(fmkv.Exception_) as e:
        book.alloc(3)
    assert e.value.code == fmkv.FMKV_ERR_CAPACITY and book.free_count() == 2
    assert book.alloc(0) == []
    book.release([a[1], -1, a[0]])
    assert book.free_count() == 4 and book.users(a[1]) == 0 and book.users(a[2]) == 1
    assert book.alloc(1) == [a[1]]  # the first one given back is the first one taken


@pytest.mark.parametrize("bad", [[0, 9], [0, -2], [0, 1, 0], [3], [0, 0]])
def test_bad_release_changes_nothing(bad):
    book = fmkv.PageBook(4)
    assert book.alloc(2) == [0, 1]
    with pytest.raises(fmkv.Exception_) as e:
        book.release(bad)
    assert e.value.code == fmkv.FMKV_ERR_INVALID_ARG
    assert book.free_count() == 2 and [book.users(b) for b in range(4)] == [1, 1, 0, 0]


def test_release_of_a_shared_block_listed_twice():
    book = fmkv.PageBook(4)
    a = book.alloc(2)
    child, copy = book.fork(a, 32)
    assert child == a and copy is None and book.users(a[0]) == 2
    book.release([a[0], a[0], a[1]])
    assert book.free_count() == 3 and book.users(a[0]) == 0 and book.users(a[1]) == 1
    assert sorted(book.alloc(3)) == sorted({0, 1, 2, 3} - {a[1]})


@pytest.mark.parametrize("n_tokens,shared", [(0, 0), (1, 0), (15, 0), (16, 1), (17, 1), (47, 2), (48, 3)])
def test_fork(n_tokens, shared):
    book = fmkv.PageBook(8)
    a = book.alloc(4)
    child, copy = book.fork(a, n_tokens)
    assert len(child) == -(-n_tokens // 16) and child[:shared] == a[:shared]
    if n_tokens % 16:
        assert copy == (a[shared], child[shared]) and child[shared] not in a and book.users(child[shared]) == 1
    else:
        assert copy is None
    assert [book.users(b) for b in a] == [2 if i < shared else 1 for i in range(4)]
    book.release(child)
    assert book.free_count() == 4 and all(book.users(b) == 1 for b in a)


def test_fork_without_room_or_of_a_free_block_changes_nothing():
    book = fmkv.PageBook(2)
    a = book.alloc(2)
    with pytest.raises(fmkv.Exception_) as e:
        book.fork(a, 20)
    assert e.value.code == fmkv.FMKV_ERR_CAPACITY and [book.users(b) for b in a] == [1, 1]
    book.release(a[1:])
    with pytest.raises(fmkv.Exception_) as e:
        book.fork(a, 32)
    assert e.value.code == fmkv.FMKV_ERR_INVALID_ARG and book.users(a[0]) == 1
    with pytest.raises(ValueError):
        book.fork(a, 33)


def test_fork_keeps_blocks_given_back():
    book = fmkv.PageBook(8)
    a = book.alloc(4)
    a = book.slide(a, 64, 17)
    assert a[:3] == [-1, -1, -1] and a[3] != -1
    child, copy = book.fork(a, 60)
    assert child[:3] == [-1, -1, -1] and copy == (a[3], child[3])


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 31, 32, 33, 40, 200])
@pytest.mark.parametrize("sinks", [0, 1, 16, 20])
def test_slide_keeps_what_later_queries_see(window, sinks):
    for n in (0, 1, 16, 33, 64, 100):
        book = fmkv.PageBook(8)
        a = book.alloc(7)
        b = book.slide(a, n, window, sinks)
        for i in range(7):
            lo, hi = 16 * i, 16 * i + 15
            hidden = lo >= sinks and hi <= n - window  # every position j <= p - window for p >= n
            assert (b[i] == -1) == hidden, (n, i)
            assert book.users(a[i]) == (0 if hidden else 1)
        assert book.slide(b, n, window, sinks) == b


def test_slide_of_shared_blocks_and_bad_ones():
    book = fmkv.PageBook(8)
    a = book.alloc(4)
    child, _ = book.fork(a, 64)
    b = book.slide(a, 64, 1)
    assert b == [-1, -1, -1, -1] and [book.users(x) for x in child] == [1] * 4 and book.free_count() == 4
    assert book.slide(child, 64, 1) == b and book.free_count() == 8
    with pytest.raises(fmkv.Exception_):
        book.slide([0, 1, 2, 3], 64, 1)  # free ones
    for window, sinks in ((0, 0), (1, -1)):
        with pytest.raises(fmkv.Exception_):
            book.slide([-1] * 4, 64, window, sinks)


def test_book_arguments():
    for n in (0, -1, 1 << 31):
        with pytest.raises(fmkv.Exception_) as e:
            fmkv.PageBook(n)
        assert e.value.code == fmkv.FMKV_ERR_INVALID_ARG
    lib = fmkv.load_library()
    assert lib.fmkv_pages_destroy(None) == fmkv.FMKV_OK
    assert lib.fmkv_pages_alloc(None, 1, None) == fmkv.FMKV_ERR_INVALID_ARG
    assert lib.fmkv_pages_release(None, None, 1) == fmkv.FMKV_ERR_INVALID_ARG
    book = fmkv.PageBook(2)
    for bad in (-1, 2):
        with pytest.raises(fmkv.Exception_):
            book.users(bad)
    with pytest.raises(fmkv.Exception_):
        book.alloc(-1)


def test_random_use_keeps_the_book():
    """Sequences that grow, fork, slide and end: users are what the sequences hold."""
    rng = random.Random(3)
    book = fmkv.PageBook(64)
    seqs = []
    for _ in range(2000):
        act = rng.random()
        try:
            if act < 0.3 or not seqs:
                n = rng.randint(1, 120)
                seqs.append([book.alloc(-(-n // 16)), n])
            elif act < 0.5:
                blocks, n = rng.choice(seqs)
                child, copy = book.fork(blocks, n)
                assert copy is None or (copy[0] in blocks and copy[1] in child)
                seqs.append([child, n])
            elif act < 0.7:
                s = rng.choice(seqs)
                s[0] = book.slide(s[0], s[1], rng.randint(1, 60), rng.choice([0, 5, 16]))
            else:
                blocks, _ = seqs.pop(rng.randrange(len(seqs)))
                book.release(blocks)
        except fmkv.Exception_ as e:
            assert e.code == fmkv.FMKV_ERR_CAPACITY
            blocks, _ = seqs.pop(rng.randrange(len(seqs)))
            book.release(blocks)
        held = [sum(blocks.count(b) for blocks, _ in seqs) for b in range(64)]
        assert held == [book.users(b) for b in range(64)]
        assert book.free_count() == held.count(0)


@pytest.mark.parametrize("wide", [2 ** 32, -2 ** 32 + 1, 2 ** 31])
def test_numbers_past_32_bits_are_refused(wide):
    book = fmkv.PageBook(8)
    a = book.alloc(4)
    for call in (lambda: book.release([a[0], wide]), lambda: book.users(wide), lambda: book.fork([wide], 5),
                 lambda: book.slide(a, 64, wide + 16), lambda: book.slide(a, 64, 16, wide),
                 lambda: book.slide([a[0], wide], 32, 16)):
        with pytest.raises(ValueError):
            call()
    assert book.free_count() == 4 and [book.users(b) for b in a] == [1] * 4


@pytest.mark.parametrize("low", [2, 16, 40, 1600])
def test_counts_past_64_bits_are_refused(low):
    """(Their low 64 bits would be counts that the buffers were not made for.)"""
    book = fmkv.PageBook(64)
    a = book.alloc(4)
    for wide in (low - 2 ** 64, low + 2 ** 64, -2 ** 63 - 1, 2 ** 63):
        for call in (lambda: fmkv.PageBook(wide), lambda: fmkv.PagedPool(fmkv.make_desc(2, 128, 4), wide),
                     lambda: book.alloc(wide), lambda: book.fork(a, wide), lambda: book.slide(a, wide, 16)):
            with pytest.raises((ValueError, fmkv.Exception_)):
                call()
    for call in (lambda: book.alloc(-5), lambda: book.fork(a, -5), lambda: book.slide(a, -5, 16)):
        with pytest.raises(fmkv.Exception_):
            call()
    assert book.free_count() == 60 and [book.users(b) for b in a] == [1] * 4


@pytest.mark.parametrize("n_tokens", [2 ** 63 - 1, 2 ** 63 - 14, 2 ** 40, 2 ** 31, -1, -2 ** 63])
def test_sequences_past_32_bit_positions_are_refused(n_tokens):
    import ctypes

    lib, book = fmkv.load_library(), fmkv.PageBook(4)
    book.alloc(2)
    blocks, child = (ctypes.c_int32 * 2)(0, 1), (ctypes.c_int32 * 2)(7, 7)
    src, dst, freed = ctypes.c_int32(5), ctypes.c_int32(5), ctypes.c_int64(5)
    assert lib.fmkv_pages_fork(book._h, blocks, n_tokens, child, ctypes.byref(src),
                               ctypes.byref(dst)) == fmkv.FMKV_ERR_INVALID_ARG
    assert lib.fmkv_pages_slide(book._h, blocks, n_tokens, 16, 0, ctypes.byref(freed)) == fmkv.FMKV_ERR_INVALID_ARG
    assert list(blocks) == [0, 1] and list(child) == [7, 7] and (src.value, dst.value, freed.value) == (5, 5, 5)
    assert [book.users(b) for b in range(4)] == [1, 1, 0, 0] and book.free_count() == 2


def test_fork_behind_the_window_is_refused():
    """A fork from a position in a block that was given back: its tokens are gone, and
    the next one would be stored nowhere."""
    book = fmkv.PageBook(8)
    a = book.slide(book.alloc(4), 64, 17)
    for n in (1, 17, 33, 47):
        with pytest.raises(fmkv.Exception_) as e:
            book.fork(a, n)
        assert e.value.code == fmkv.FMKV_ERR_INVALID_ARG
    assert book.free_count() == 7 and book.users(a[3]) == 1
    assert book.fork(a, 48) == ([-1, -1, -1], None)
