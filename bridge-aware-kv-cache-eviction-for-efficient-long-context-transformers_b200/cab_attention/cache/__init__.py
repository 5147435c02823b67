from .paged import PagedKVCache  # noqa: F401
