"""The package's error type."""


class PagedAttentionError(RuntimeError):
    """PagedAttentionError / KVCacheError text from pam_last_error."""
