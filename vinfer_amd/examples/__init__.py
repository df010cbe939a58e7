"""Small programs that use the package as a caller does."""
